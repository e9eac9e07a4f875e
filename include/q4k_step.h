/*
 * q4k_step.h -- C ABI of the operators that a decode step needs between its
 * projections (q4k_gemv.h) and its next token (MI355X, gfx950):
 *   q4k_rope        norms of queries and keys for each head and the rotation by
 *                   their positions, in one pass
 *   q4k_kv8_store   new keys and values into a paged cache of 8 bits with a scale
 *                   for each block of tokens and head
 *   q4k_kv8_load    tokens of such a cache as the values they stand for
 *   q4k_kv8_attn    attention of a batch of requests over such a cache
 *   q4k_sample      the next tokens from logits: temperature, top-k, top-p, min-p
 *                   and given random numbers
 * No counterpart in the reference, whose path ends at the product.
 *
 * Conventions as in q4k_batch.h: strides (nb*) in bytes, a q4k_status, device
 * work on the caller's HIP stream without host synchronisation, nothing thrown
 * or aborted, descriptors read during the call; what the device reads
 * (positions, lengths, page tables, sampling rules) may change between replays
 * of a captured graph, entries out of range are ignored as each call states.
 * Equal calls give equal bits.  A workspace needs no initial contents and may be
 * used by any call that the stream orders after the last one, by one at a time.
 * A call that would take 2^32 threads and more in a launch (64 a token of q4k_rope,
 * 512 a row of q4k_sample, one for eight values that n_requests times n_q tokens
 * would have in q4k_kv8_load) is refused with Q4K_EUNSUPPORTED as a whole.
 */
#ifndef Q4K_STEP_H
#define Q4K_STEP_H

#include "q4k_batch.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------- norms and rotation of queries and keys */

#define Q4K_ROPE_MAX_HEAD_DIM 256
#define Q4K_ROPE_NORMAL 0 /* pairs of neighbours, (2i, 2i + 1) (GGML_ROPE_TYPE_NORMAL) */
#define Q4K_ROPE_NEOX 2   /* pairs of halves, (i, i + n_rot / 2) (GGML_ROPE_TYPE_NEOX) */

/* Rows of one kind, the queries or the keys: n_head heads a token. */
typedef struct q4k_rope_rows {
    const void *src;
    void *dst;         /* may be src with its type and strides, else must not overlap it */
    int32_t src_type;  /* Q4K_GGML_TYPE_F32, _F16 or _BF16 */
    int32_t dst_type;  /* src_type; for F32 also F16 or BF16 */
    int64_t n_head;
    int64_t nb_src_token, nb_src_head, nb_dst_token, nb_dst_head;
    const float *norm; /* head_dim factors on the device: y = x / sqrt(mean(x^2) + eps) * norm
                        * over each head first; NULL: none */
} q4k_rope_rows;

typedef struct q4k_rope_args {
    int32_t head_dim; /* even, up to Q4K_ROPE_MAX_HEAD_DIM */
    int32_t n_rot;    /* the first n_rot dimensions are rotated (even, 0..head_dim), the others passed on */
    int32_t mode;     /* Q4K_ROPE_NORMAL or Q4K_ROPE_NEOX */
    float eps;
    /* Pair i turns by pos * freq_base^(-2i / n_rot) / freq_factors[i] * s_i, with s_i =
     * freq_scale, or where ext_factor is not 0 (YaRN) freq_scale (1 - r_i) + r_i,
     * r_i = ext_factor * (1 - clamp((i - lo) / max(0.001, hi - lo), 0, 1)), lo and hi
     * the pairs that turn beta_fast and beta_slow times over n_ctx_orig positions
     * (rounded down and up, within 0..n_rot - 1); results are multiplied by attn_factor,
     * with ext_factor also by 1 + 0.1 ln(1 / freq_scale). */
    float freq_base, freq_scale, ext_factor, attn_factor, beta_fast, beta_slow;
    int64_t n_ctx_orig;
    const float *freq_factors; /* n_rot / 2 on the device, NULL: 1 */
    int64_t n_tokens;
    const int32_t *pos; /* n_tokens positions on the device, of any value */
    const q4k_rope_rows *q, *k; /* either may be NULL */
} q4k_rope_args;

/* Angles are worked out in 64 bits and reduced before they are rounded; norms and
 * rotations are F32, results are rounded once.  Rows of 16-byte aligned addresses
 * and strides, with n_rot / 2 and head_dim - n_rot multiples of 4 and 8, run faster. */
int q4k_rope(const q4k_rope_args *args, void *stream);

/* ------------------------------------- keys and values in 8 bits, paged */

#define Q4K_TYPE_I8 24     /* GGML_TYPE_I8: -127..127 times the scale */
#define Q4K_TYPE_E4M3 1000 /* OCP 8-bit floats of 4 exponent bits, up to 448, times the scale (no ggml type) */

#define Q4K_KV8_MAX_HEAD_DIM 256

/* Keys and values in pages of page_size tokens, one byte a value: token t of head
 * h in page p is at k + p * nb_k_page + t * nb_k_token + h * nb_k_head, head_dim
 * contiguous values (v alike), and stands for its values times the scale at
 * k_scale + p * nb_s_page + (t / block) * nb_s_block + h * nb_s_head (v_scale
 * alike, with the same strides).  page_size is a multiple of block.  k, v and
 * their strides are multiples of 16 bytes, else Q4K_EUNSUPPORTED. */
typedef struct q4k_kv8_pages {
    int32_t type;  /* Q4K_TYPE_I8 or Q4K_TYPE_E4M3 */
    int32_t n_head_kv, head_dim; /* head_dim: a multiple of 16 up to Q4K_KV8_MAX_HEAD_DIM */
    int32_t block; /* tokens of a scale */
    void *k, *v;   /* (only q4k_kv8_store writes) */
    int64_t n_pages, page_size;
    int64_t nb_k_page, nb_k_token, nb_k_head;
    int64_t nb_v_page, nb_v_token, nb_v_head;
    float *k_scale, *v_scale;
    int64_t nb_s_page, nb_s_block, nb_s_head;
    /* page numbers as in q4k_kv_pages; NULL: pages r * table_len, r * table_len + 1, ... */
    const int32_t *table;
    int64_t table_stride, table_len;
} q4k_kv8_pages;

/* The last tokens of each request: with len = len[r] and n tokens, token t of
 * request r has position len - n + t. */
typedef struct q4k_kv8_rows {
    const q4k_kv8_pages *pages;
    int32_t type;           /* of k and v here: Q4K_GGML_TYPE_F32, _F16 or _BF16 */
    int64_t n_tokens, n_requests;
    int64_t n_q;            /* tokens of each request, with q_start the most of any */
    const int32_t *q_start; /* as in q4k_prefix_attn_args; NULL: r * n_q */
    const int32_t *len;     /* device, n_requests, clamped to 0..max_len */
    int64_t max_len;        /* up to 2^30 */
    void *k, *v;            /* n_tokens rows of n_head_kv heads of head_dim (q4k_kv8_store: read only) */
    int64_t nb_k_token, nb_k_head, nb_v_token, nb_v_head;
} q4k_kv8_rows;

/* Writes each request's new tokens into its pages.  A block's scale becomes the
 * largest magnitude of its new tokens / 127 (E4M3: / 448), or stays what it is
 * where the block holds earlier tokens of the request and their scale is larger;
 * where it grows, the earlier tokens are rounded again from the values that they
 * stood for (in F32).  Values are the nearest to x / scale, ties to even (worked out
 * exactly).  Infinities and NaN take no part in the magnitude; infinities become the
 * largest of their sign (of a scale of 1 where the block's would be 0), NaN 0.
 * Tokens at positions below 0 or in pages out of range are left out, bytes of
 * positions that no new or earlier token of the block has stay as they are.  Two
 * requests' new tokens must not fall into one block, nor a block of one hold earlier
 * tokens of another that is read meanwhile.  Pages, tokens, heads and scales that overlap
 * (a stride of 0, say, which q4k_kv8_load and q4k_kv8_attn take) are Q4K_EINVAL. */
int q4k_kv8_store(const q4k_kv8_rows *rows, void *stream);

/* Reads each request's last tokens as the values they stand for (byte times scale in
 * F32, then rounded to `type`): zeros at positions below 0 and in pages out of range.  Rows of no
 * request stay as they are.  k or v may be NULL. */
int q4k_kv8_load(const q4k_kv8_rows *rows, void *stream);

typedef struct q4k_kv8_attn_args {
    const q4k_kv8_pages *pages;
    int32_t q_type;  /* of q and dst: Q4K_GGML_TYPE_F32, _F16 or _BF16 */
    int32_t n_head;  /* a multiple of pages->n_head_kv */
    float scale;     /* factor of q.k, usually head_dim^-0.5 */
    int64_t n_tokens, n_requests;
    int64_t n_q;            /* as in q4k_kv8_rows */
    const int32_t *q_start;
    const int32_t *len;
    int64_t max_len;
    const void *q;
    int64_t nb_q_token, nb_q_head;
    void *dst;
    int64_t nb_dst_token, nb_dst_head;
    float *lse; /* n_tokens x n_head, as in q4k_prefix_attn_args; may be NULL */
} q4k_kv8_attn_args;

/* Bytes of workspace that q4k_kv8_attn takes (0 if the arguments are invalid or
 * it takes none). */
size_t q4k_kv8_attn_workspace_bytes(const q4k_kv8_attn_args *args);

/* Attention of every request's last tokens over the request's tokens: token t of n
 * sees positions up to len - n + t.  What a query does not see has no effect on
 * it; one that sees nothing gives zeros and an lse of -inf; tokens of no request
 * are left as they are.  Scores, the softmax's maximum and sum and the output sum
 * are F32.  Bytes enter the matrix cores exactly, as F16 (keys; BF16 with BF16
 * queries) and BF16 (values), scales are applied in F32; queries of F32 enter as
 * two F16 values (22 bits, or 2^-39 of the head's largest value), probabilities times
 * their value's scale as three BF16 values with F32 queries and two with queries of
 * 16 bits.  Scales of keys below 2^96, of values below 2^100.  dst and lse must not overlap what is read.  max_len / 128 times the KV heads
 * times a request's tiles of 16 rows stays below 2^31, else Q4K_EUNSUPPORTED. */
int q4k_kv8_attn(const q4k_kv8_attn_args *args, void *workspace, size_t workspace_bytes, void *stream);

/* ---------------------------------------------------------- next tokens */

/* Per-row rules on the device, n_rows each; absent ones are NULL. */
typedef struct q4k_sample_rules {
    const float *temperature; /* NULL: 1; 0 and below, or NaN: the largest logit */
    const int32_t *top_k;     /* 0 and below: all */
    const float *top_p;       /* 1 and above, or NaN: all */
    const float *min_p;       /* 0 and below, or NaN: all; 1 and above: 1 */
    const float *uniform;     /* in [0, 1) (clamped to it, NaN: 0); NULL: the largest logit of every row */
} q4k_sample_rules;

/* Bytes of workspace that are enough for q4k_sample of these sizes and of any
 * smaller n_rows (0: invalid sizes, or none taken). */
size_t q4k_sample_workspace_bytes(int64_t n_vocab, int64_t n_rows);

/* tokens[i] = a token of row i of src (F32, n_rows rows of up to 2^30 n_vocab
 * logits).  With m the row's largest logit, w_v = exp((l_v - m) / temperature); the
 * cuts, one after the other:
 *   top-k   the top_k largest logits (of equal ones the lower tokens)
 *   top-p   of those, in descending order (of equal ones the lower tokens first), each
 *           whose predecessors' sum of w is below top_p times the sum of all of
 *           them, and always the first
 *   min-p   of those, w_v >= min_p
 * The token is the first, in the order of token numbers, up to which the kept w's
 * sum exceeds uniform times their sum.  Logits of -inf and NaN are no candidates; a
 * row without any gives -1; with logits of +inf those are the candidates, alike.
 * w and its sums are 64 bits; sums within 2^-40 of a border (of its own value) count as
 * equal to it, tokens below 2^-63 of the largest w as 0.
 * logprob[i] (may be NULL): the logarithm of the token's share of the kept
 * w's sum, 0 where the largest logit was taken, -inf where there is none. */
int q4k_sample(const float *src, int64_t n_vocab, int64_t n_rows, int64_t nb_src, const q4k_sample_rules *rules,
               int32_t *tokens, float *logprob, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif

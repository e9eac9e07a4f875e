/*
 * q4k_batch.h -- C ABI of the operators that a batch of requests decoded
 * together needs beside the quantised products of q4k_gemv.h (MI355X, gfx950):
 *   q4k_lora_add       low-rank adapters, one per token, added to the result of
 *                      a projection that all tokens share
 *   q4k_prefix_attn    attention over a prefix that all requests share, read
 *                      once for all of them, and each request's own tokens
 *   q4k_logits_adjust  penalties for repeated tokens, biases and grammar masks
 *                      on the output projection's logits
 * No counterpart in the reference, whose path ends at the product.
 *
 * Conventions as in q4k_gemv.h: plain pointers and sizes, strides (nb*) in
 * bytes, a q4k_status, device work on the caller's HIP stream without host
 * synchronisation, nothing thrown or aborted.  Descriptors are read during the
 * call and not kept.  What the device reads (ids, lengths, page tables, list
 * starts) may change between calls and between replays of a captured graph;
 * entries out of range are ignored as each call states, never followed.
 * Outputs do not depend on the order in which workgroups run: equal calls give
 * equal bits.  A workspace needs no initial contents and may be used by any
 * call that the stream orders after the last one; without one the call takes a
 * stream-ordered temporary (hipMallocAsync), which a capturing caller avoids.
 */
#ifndef Q4K_BATCH_H
#define Q4K_BATCH_H

#include "q4k_gemv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define Q4K_GGML_TYPE_F16 1
#define Q4K_GGML_TYPE_BF16 30

/* ---------------------------------------------------- low-rank adapters */

#define Q4K_LORA_MAX_RANK 256

/* The adapters of one projection of ne01 rows of ne00 weights.  Adapter i is
 * a[i] (rank rows of ne00 values) and b[i] (ne01 rows of rank values), both F16
 * or BF16: the layouts of a GGUF adapter file's lora_a and lora_b tensors. */
typedef struct q4k_lora {
    int32_t type;          /* Q4K_GGML_TYPE_F16 or Q4K_GGML_TYPE_BF16 */
    int32_t rank;          /* values of a row of b, 1..Q4K_LORA_MAX_RANK */
    int64_t n_adapters;
    const void *a;
    int64_t nb_a, nb_a_adapter; /* bytes from a row to the next, from an adapter to the next */
    const void *b;
    int64_t nb_b, nb_b_adapter;
    const float *scale;    /* n_adapters factors on the device (alpha / rank), NULL = 1 */
    const int32_t *ranks;  /* n_adapters ranks on the device: only the first ranks[i] rows of a[i]
                            * and columns of b[i] count (clamped to 0..rank); NULL = rank */
} q4k_lora;

/* Bytes of workspace that are enough for q4k_lora_add of ne11 tokens and of any
 * fewer (0: invalid sizes). */
size_t q4k_lora_workspace_bytes(const q4k_lora *lora, int64_t ne00, int64_t ne01, int64_t ne11);

/* dst[n] = src2[n] + scale[i] * b[i] (a[i] src1[n]),  i = ids[n], for n < ne11.
 *   src1: ne11 tokens of ne00 floats, token stride nb11 bytes
 *   src2: ne11 tokens of ne01 floats (the shared projection's result), stride
 *         nb21; NULL = zeros; may be dst itself (same stride), else must not
 *         overlap it
 *   ids:  ne11 adapter numbers on the device; a token whose number is outside
 *         [0, n_adapters) takes no adapter: dst[n] = src2[n]
 *   dst:  ne11 tokens of ne01 floats, stride nb1
 * Any ne01, ne11 and rank, ne00 up to 2^30; rows of a and b that are 16-byte
 * aligned and rows of dst that are 64-byte aligned run faster.  Sums are F32; the
 * F32 activations and a's products enter the matrix cores as sums of three BF16
 * values, which hold F32's 24 bits; an activation or sum that is not finite in
 * BF16 (past 3.39e38) makes its token's results NaN.  With ne00 == 0 or a rank of 0
 * an adapter adds nothing, whatever its scale and values. */
int q4k_lora_add(const q4k_lora *lora, int64_t ne00, int64_t ne01, const float *src1, int64_t ne11,
                 int64_t nb11, const int32_t *ids, const float *src2, int64_t nb21, float *dst,
                 int64_t nb1, void *workspace, size_t workspace_bytes, void *stream);

/* ---------------------------------------------- shared-prefix attention */

#define Q4K_ATTN_MAX_HEAD_DIM 256

/* Keys and values in pages of page_size tokens: token t of head h in page p is
 * at k + p * nb_k_page + t * nb_k_token + h * nb_k_head, head_dim contiguous
 * values (v alike).  k, v and their strides are multiples of 16 bytes, else
 * Q4K_EUNSUPPORTED.  A contiguous cache is one page. */
typedef struct q4k_kv_pages {
    const void *k, *v;
    int64_t n_pages, page_size;
    int64_t nb_k_page, nb_k_token, nb_k_head;
    int64_t nb_v_page, nb_v_token, nb_v_head;
    /* Page numbers on the device: table_len of them in the order of the tokens,
     * for request r from table + r * table_stride (the prefix: from table).
     * NULL: pages r * table_len, r * table_len + 1, ...  Tokens of a page
     * outside [0, n_pages) are not seen. */
    const int32_t *table;
    int64_t table_stride, table_len;
} q4k_kv_pages;

typedef struct q4k_prefix_attn_args {
    int32_t q_type;   /* of q and dst: Q4K_GGML_TYPE_F32 or kv_type */
    int32_t kv_type;  /* Q4K_GGML_TYPE_F16 or Q4K_GGML_TYPE_BF16 */
    int32_t n_head, n_head_kv, head_dim; /* n_head a multiple of n_head_kv; head_dim a multiple of
                                          * 8 up to Q4K_ATTN_MAX_HEAD_DIM */
    float scale;                         /* factor of q.k, usually head_dim^-0.5 */
    int64_t n_tokens, n_requests;
    int64_t n_q;            /* tokens of each request, with q_start the most of any request */
    const int32_t *q_start; /* device, n_requests + 1: request r has the tokens [q_start[r],
                             * q_start[r+1]), clamped to n_tokens and to n_q of them; NULL: r * n_q */
    const void *q;
    int64_t nb_q_token, nb_q_head;
    const q4k_kv_pages *prefix; /* n_prefix tokens that every query sees; NULL if n_prefix is 0 */
    int64_t n_prefix;
    const q4k_kv_pages *suffix;  /* each request's own tokens; NULL if max_suffix is 0 */
    const int32_t *suffix_len;   /* device, n_requests, clamped to 0..max_suffix; NULL if max_suffix is 0 */
    int64_t max_suffix;
    void *dst;
    int64_t nb_dst_token, nb_dst_head;
    float *lse; /* n_tokens x n_head, natural logarithm of each row's sum of exponentials; may be NULL */
} q4k_prefix_attn_args;

/* Bytes of workspace that q4k_prefix_attn takes (0 if the arguments are
 * invalid or it takes none). */
size_t q4k_prefix_attn_workspace_bytes(const q4k_prefix_attn_args *args);

/* Attention of every request's tokens over the shared prefix and the request's
 * own tokens, whose last ones are the queries' own: with len = suffix_len[r]
 * and n queries, query t of request r sees own positions up to len - n + t (a
 * negative bound: none).  A query that sees nothing gives zeros and an lse of
 * -inf.  Values and keys that a query does not see, and memory past the
 * lengths, have no effect on it whatever they hold.  Scores, the softmax's
 * maximum and sum and the output sum are F32.  With q_type F32 the queries and
 * probabilities enter the matrix cores as sums of two (F16) or three (BF16)
 * values of kv_type, with q_type kv_type as one rounded value.  Tokens of no
 * request (before, between and behind those that q_start names, or past n_q of a
 * request) are left as they are.  dst and lse must not overlap what is read.  Up
 * to 2^30 positions a part. */
int q4k_prefix_attn(const q4k_prefix_attn_args *args, void *workspace, size_t workspace_bytes,
                    void *stream);

/* -------------------------------------- penalties, biases, masks on logits */

/* What changes the logits of each row; absent parts are NULL. */
typedef struct q4k_logits_rules {
    /* per-row factors on the device, n_rows each */
    const float *repeat;    /* logits of tokens in the row's history: divided by it if > 0, else multiplied */
    const float *frequency; /* subtracted once per occurrence in the history */
    const float *presence;  /* subtracted once from every token in the history */
    /* the rows' histories one after the other: row i has the entries
     * [history_start[i], history_start[i+1]), clamped to n_history (and to less
     * than 2^31 of them) */
    const int32_t *history;
    const int64_t *history_start;
    int64_t n_history;
    /* biases, alike: bias[j] is added to token bias_ids[j]; of several entries
     * of a token in a row the last one counts */
    const int32_t *bias_ids;
    const float *bias;
    const int64_t *bias_start;
    int64_t n_bias;
    /* bit v % 32 of word v / 32 of a mask row is 1 where token v is allowed;
     * others become -inf.  Row i has mask row mask_rows[i] (none if outside
     * [0, n_masks)); mask_rows NULL: row i, which needs n_masks >= n_rows */
    const int32_t *mask;
    int64_t n_masks, nb_mask;
    const int32_t *mask_rows;
} q4k_logits_rules;

/* dst = src (F32, n_rows rows of up to 2^30 n_vocab logits) with, per row and in this
 * order: the repetition factor, frequency and presence penalties, biases, the
 * mask.  Token ids outside [0, n_vocab) are ignored.  dst may be src (same
 * stride), else must not overlap it.  Takes no workspace. */
int q4k_logits_adjust(const float *src, int64_t n_vocab, int64_t n_rows, int64_t nb_src,
                      const q4k_logits_rules *rules, float *dst, int64_t nb_dst, void *stream);

#ifdef __cplusplus
}
#endif
#endif

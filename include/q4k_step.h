/*
 * q4k_step.h -- C ABI of the operators that a decode step needs between its
 * projections (q4k_gemv.h) and its next token (MI355X, gfx950):
 *   q4k_rope        norms of queries and keys for each head and the rotation by
 *                   their positions, in one pass
 * No counterpart in the reference, whose path ends at the product.
 *
 * Conventions as in q4k_batch.h: strides (nb*) in bytes, a q4k_status, device
 * work on the caller's HIP stream without host synchronisation, nothing thrown
 * or aborted, descriptors read during the call; what the device reads
 * (positions, lengths, page tables, sampling rules) may change between replays
 * of a captured graph, entries out of range are ignored as each call states.
 * Equal calls give equal bits.  A workspace needs no initial contents and may be
 * used by any call that the stream orders after the last one, by one at a time.
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

#ifdef __cplusplus
}
#endif
#endif

// q4k_kv8.h -- what the operators on paged caches of 8 bits share
// (include/q4k_step.h): the cache as kernels see it, the tokens of a request, and
// the argument checks.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/q4k_step.h"
#include "q4k_batch.h"
#include "q4k_device.h"

namespace q4k {

struct Kv8Cache {
    char *k, *v;
    float *k_scale, *v_scale;
    int64_t k_page, k_token, k_head, v_page, v_token, v_head, s_page, s_block, s_head;  // bytes
    const int32_t *table;
    int64_t table_stride;
    int n_pages, table_len;
    FastDiv page, block;  // tokens of a page and of a scale
};

// The tokens of each request: the last ones of its len.
struct Kv8Tokens {
    const int32_t *q_start, *len;
    int n_tokens, n_requests, n_q, max_len;
};

__device__ __forceinline__ void kv8_tokens(const Kv8Tokens &p, int r, int &t0, int &t1, int &len) {
    int64_t a = (int64_t)r * p.n_q, b = a + p.n_q;
    if (p.q_start) {
        a = p.q_start[r];
        b = p.q_start[r + 1];
        if (a < 0) a = 0;
        if (b > p.n_tokens) b = p.n_tokens;
        if (b > a + p.n_q) b = a + p.n_q;
        if (b < a) b = a;
    }
    t0 = (int)a;
    t1 = (int)b;
    const int n = p.len[r];
    len = n < 0 ? 0 : n > p.max_len ? p.max_len : n;
}
// The page that holds position t of request r; out of range where there is none.
__device__ __forceinline__ int kv8_page(const Kv8Cache &c, int r, int t) {
    const int e = (int)fastdiv((uint32_t)t, c.page);
    return c.table ? c.table[r * c.table_stride + e] : r * c.table_len + e;
}

// A page table as the kernels index it, for `rows` requests of up to `tokens` tokens.
inline bool kv8_pages_ok(const q4k_kv8_pages &c, int64_t tokens, int64_t rows) {
    if (!c.k || !c.v || !c.k_scale || !c.v_scale || c.n_pages < 1 || c.n_pages > INT32_MAX || c.page_size < 1 || c.page_size > INT32_MAX)
        return false;
    if (c.page_size % c.block != 0 || c.table_len < 0 || c.table_len > INT32_MAX) return false;
    if (!aligned(c.k_scale, 4) || !aligned(c.v_scale, 4) || ((c.nb_s_page | c.nb_s_block | c.nb_s_head) & 3) || !aligned(c.table, 4)) return false;
    if (c.table_len * c.page_size < tokens) return false;
    return c.table ? rows <= 1 || c.table_stride >= 0 : c.table_len <= c.n_pages / rows;
}
inline bool kv8_kind_ok(const q4k_kv8_pages &c) {
    return (c.type == Q4K_TYPE_I8 || c.type == Q4K_TYPE_E4M3) && c.n_head_kv >= 1 && c.head_dim >= 1 && c.block >= 1;
}
inline bool kv8_pages_vec(const q4k_kv8_pages &c) {
    return aligned(c.k, 16) && aligned(c.v, 16) && c.head_dim % 16 == 0 && c.head_dim <= Q4K_KV8_MAX_HEAD_DIM &&
           ((c.nb_k_page | c.nb_k_token | c.nb_k_head | c.nb_v_page | c.nb_v_token | c.nb_v_head) & 15) == 0;
}
// Q4K_OK, or why the tokens are refused; `empty` where there are none.
inline int kv8_tokens_check(int64_t n_tokens, int64_t n_requests, int64_t n_q, const int32_t *q_start, const int32_t *len, int64_t max_len,
                            bool &empty) {
    empty = false;
    if (n_tokens < 0 || n_requests < 0 || n_q < 0 || max_len < 0 || n_tokens > INT32_MAX || n_requests > INT32_MAX || n_q > INT32_MAX)
        return Q4K_EINVAL;
    if (!q_start && n_tokens != n_requests * n_q) return Q4K_EINVAL;
    if (!aligned(q_start, 4) || !aligned(len, 4)) return Q4K_EINVAL;
    empty = n_tokens == 0 || n_requests == 0 || n_q == 0;
    if (!empty && !len) return Q4K_EINVAL;
    if (max_len > (1 << 30) || (!empty && n_requests > INT32_MAX / n_q)) return Q4K_EUNSUPPORTED;
    return Q4K_OK;
}
inline Kv8Cache kv8_cache(const q4k_kv8_pages &c) {
    return Kv8Cache{(char *)c.k, (char *)c.v, c.k_scale, c.v_scale, c.nb_k_page, c.nb_k_token, c.nb_k_head, c.nb_v_page, c.nb_v_token,
                    c.nb_v_head, c.nb_s_page, c.nb_s_block, c.nb_s_head, c.table, c.table_stride, (int)c.n_pages, (int)c.table_len,
                    fastdiv_init((uint32_t)c.page_size), fastdiv_init((uint32_t)c.block)};
}

}  // namespace q4k

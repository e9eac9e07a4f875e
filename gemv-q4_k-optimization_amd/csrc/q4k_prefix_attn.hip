// q4k_prefix_attn.hip -- q4k_prefix_attn (include/q4k_batch.h): attention of a
// batch of requests over a prefix that they share and over their own tokens.
//
// For a query row (token t, head h) with scores s_j = scale * q.k_j over the
// positions j that it sees: m = max s_j, l = sum exp(s_j - m),
// out = sum exp(s_j - m) v_j / l, lse = m + ln l, in one pass over the keys with
// a running maximum and sum.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "q4k_batch_host.h"
#include "q4k_device.h"

namespace q4k {

struct AttnParams {
    q4k_prefix_attn_args a;
    q4k_kv_pages pre, suf;
};

// The element offset in bytes of token t, or -1 where its page is out of range.
__device__ __forceinline__ int64_t page_of(const q4k_kv_pages &c, int64_t r, int64_t t, int64_t &slot) {
    const int64_t e = t / c.page_size;
    slot = t - e * c.page_size;
    const int64_t pg = c.table ? (int64_t)c.table[r * c.table_stride + e] : r * c.table_len + e;
    return pg >= 0 && pg < c.n_pages ? pg : -1;
}

// One wave per query row: 64 positions at a time, a lane's dot product each,
// then their values one after the other with the head's dimensions over the
// lanes.
template <class T, class QT>
__global__ __launch_bounds__(64) void prefix_attn_kernel(AttnParams p) {
    __shared__ float qs[Q4K_ATTN_MAX_HEAD_DIM];
    const q4k_prefix_attn_args &a = p.a;
    const int lane = threadIdx.x;
    const int64_t r = blockIdx.x / a.n_q, t = blockIdx.x % a.n_q;
    const int head = blockIdx.y, hkv = head / (a.n_head / a.n_head_kv);
    int64_t tok0 = r * a.n_q, tok1 = tok0 + a.n_q;
    if (a.q_start) {
        tok0 = a.q_start[r];
        tok1 = a.q_start[r + 1];
        if (tok0 < 0) tok0 = 0;
        if (tok1 > a.n_tokens) tok1 = a.n_tokens;
        if (tok1 > tok0 + a.n_q) tok1 = tok0 + a.n_q;
    }
    const int64_t tok = tok0 + t;
    if (tok >= tok1) return;
    const QT *q = reinterpret_cast<const QT *>((const char *)a.q + tok * a.nb_q_token + head * a.nb_q_head);
    for (int d = lane; d < a.head_dim; d += 64) qs[d] = (float)q[d];
    __syncthreads();
    float m = -__builtin_inff(), l = 0.0f;
    float o[Q4K_ATTN_MAX_HEAD_DIM / 64] = {};
    for (int part = 0; part < 2; ++part) {
        const q4k_kv_pages &c = part ? p.suf : p.pre;
        int64_t len = a.n_prefix;
        if (part) {
            len = a.max_suffix > 0 ? a.suffix_len[r] : 0;
            if (len > a.max_suffix) len = a.max_suffix;
            len = len - (tok1 - tok0) + t + 1;
        }
        for (int64_t j0 = 0; j0 < len; j0 += 64) {
            const int64_t j = j0 + lane;
            int64_t slot = 0, pg = -1;
            if (j < len) pg = page_of(c, part ? r : 0, j, slot);
            float s = -__builtin_inff();
            if (pg >= 0) {
                const T *k = reinterpret_cast<const T *>((const char *)c.k + pg * c.nb_k_page + slot * c.nb_k_token +
                                                         hkv * c.nb_k_head);
                s = 0.0f;
                for (int d = 0; d < a.head_dim; ++d) s += qs[d] * (float)k[d];
                s *= a.scale;
            }
            float top = s;
            for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
            const float mn = fmaxf(m, top);
            if (mn == -__builtin_inff()) continue;
            const float w = s == -__builtin_inff() ? 0.0f : __expf(s - mn), f = __expf(m - mn);
            float sum = w;
            for (int x = 1; x < 64; x *= 2) sum += __shfl_xor(sum, x);
            l = l * f + sum;
            m = mn;
            for (int e = 0; e < Q4K_ATTN_MAX_HEAD_DIM / 64; ++e) o[e] *= f;
            for (int y = 0; y < 64; ++y) {
                const int64_t pgy = __shfl((int)pg, y);
                if (pgy < 0) continue;
                const int64_t sy = __shfl((int)slot, y);
                const float wy = __shfl(w, y);
                const T *v = reinterpret_cast<const T *>((const char *)c.v + pgy * c.nb_v_page + sy * c.nb_v_token +
                                                         hkv * c.nb_v_head);
                for (int e = 0; e < Q4K_ATTN_MAX_HEAD_DIM / 64; ++e)
                    if (e * 64 + lane < a.head_dim) o[e] += wy * (float)v[e * 64 + lane];
            }
        }
    }
    QT *out = reinterpret_cast<QT *>((char *)a.dst + tok * a.nb_dst_token + head * a.nb_dst_head);
    for (int e = 0; e < Q4K_ATTN_MAX_HEAD_DIM / 64; ++e)
        if (e * 64 + lane < a.head_dim) out[e * 64 + lane] = (QT)(l == 0.0f ? 0.0f : o[e] / l);
    if (a.lse && lane == 0) a.lse[tok * a.n_head + head] = l == 0.0f ? -__builtin_inff() : m + logf(l);
}

static bool pages_ok(const q4k_kv_pages &c, int64_t tokens, int64_t rows) {
    if (!c.k || !c.v || c.n_pages < 1 || c.n_pages > INT32_MAX || c.page_size < 1 || c.page_size > INT32_MAX) return false;
    if (!aligned(c.k, 2) || !aligned(c.v, 2) || !aligned(c.table, 4) || c.table_len < 0 || c.table_len > INT32_MAX) return false;
    if (c.table_len * c.page_size < tokens) return false;
    if (c.table ? rows > 1 && c.table_stride < 0 : c.table_len > c.n_pages / rows) return false;
    return true;
}
static bool pages_vec(const q4k_kv_pages &c) {
    return aligned(c.k, 16) && aligned(c.v, 16) &&
           ((c.nb_k_page | c.nb_k_token | c.nb_k_head | c.nb_v_page | c.nb_v_token | c.nb_v_head) & 15) == 0;
}

// Q4K_OK with empty set where there is nothing to do
static int attn_check(const q4k_prefix_attn_args *args, bool &empty) {
    if (!args) return Q4K_EINVAL;
    const q4k_prefix_attn_args &a = *args;
    empty = false;
    if (a.kv_type != Q4K_GGML_TYPE_F16 && a.kv_type != Q4K_GGML_TYPE_BF16) return Q4K_EINVAL;
    if (a.q_type != Q4K_GGML_TYPE_F32 && a.q_type != a.kv_type) return Q4K_EINVAL;
    if (a.n_head < 1 || a.n_head_kv < 1 || a.n_head % a.n_head_kv != 0 || a.head_dim < 1) return Q4K_EINVAL;
    if (a.n_tokens < 0 || a.n_requests < 0 || a.n_q < 0 || a.n_prefix < 0 || a.max_suffix < 0) return Q4K_EINVAL;
    if (a.n_tokens > INT32_MAX || a.n_requests > INT32_MAX || a.n_q > INT32_MAX || a.n_prefix > INT32_MAX ||
        a.max_suffix > INT32_MAX)
        return Q4K_EINVAL;
    if (!a.q_start && a.n_tokens != a.n_requests * a.n_q) return Q4K_EINVAL;
    if (a.n_tokens == 0 || a.n_requests == 0 || a.n_q == 0) {
        empty = true;
        return Q4K_OK;
    }
    const int es = a.q_type == Q4K_GGML_TYPE_F32 ? 4 : 2;
    if (!a.q || !a.dst || !aligned(a.q, es) || !aligned(a.dst, es) || !aligned(a.lse, 4) || !aligned(a.q_start, 4))
        return Q4K_EINVAL;
    if (a.nb_q_token % es != 0 || a.nb_q_head % es != 0 || a.nb_dst_token % es != 0 || a.nb_dst_head % es != 0)
        return Q4K_EINVAL;
    if ((a.n_head > 1 && (a.nb_q_head < es * (int64_t)a.head_dim || a.nb_dst_head < es * (int64_t)a.head_dim))) return Q4K_EINVAL;
    if (a.n_prefix > 0 && (!a.prefix || !pages_ok(*a.prefix, a.n_prefix, 1))) return Q4K_EINVAL;
    if (a.max_suffix > 0 &&
        (!a.suffix || !a.suffix_len || !aligned(a.suffix_len, 4) || !pages_ok(*a.suffix, a.max_suffix, a.n_requests)))
        return Q4K_EINVAL;
    if (a.head_dim % 8 != 0 || a.head_dim > Q4K_ATTN_MAX_HEAD_DIM) return Q4K_EUNSUPPORTED;
    if ((a.n_prefix > 0 && !pages_vec(*a.prefix)) || (a.max_suffix > 0 && !pages_vec(*a.suffix))) return Q4K_EUNSUPPORTED;
    if (a.n_requests * a.n_q > INT32_MAX || a.n_head > 65535) return Q4K_EUNSUPPORTED;
    return Q4K_OK;
}

}  // namespace q4k

using namespace q4k;

extern "C" {

size_t q4k_prefix_attn_workspace_bytes(const q4k_prefix_attn_args *) { return 0; }

int q4k_prefix_attn(const q4k_prefix_attn_args *args, void *workspace, size_t workspace_bytes, void *stream) {
    bool empty;
    int st = attn_check(args, empty);
    if (st != Q4K_OK || empty) return st;
    DeviceInfo *di;
    st = device_info(&di);
    if (st != Q4K_OK) return st;
    (void)workspace;
    (void)workspace_bytes;
    AttnParams p{*args, {}, {}};
    if (p.a.n_prefix > 0) p.pre = *p.a.prefix;
    if (p.a.max_suffix > 0) p.suf = *p.a.suffix;
    const bool f32 = p.a.q_type == Q4K_GGML_TYPE_F32;
    auto *fn = p.a.kv_type == Q4K_GGML_TYPE_F16
                   ? (f32 ? prefix_attn_kernel<_Float16, float> : prefix_attn_kernel<_Float16, _Float16>)
                   : (f32 ? prefix_attn_kernel<__hip_bfloat16, float> : prefix_attn_kernel<__hip_bfloat16, __hip_bfloat16>);
    return launch(fn, dim3((unsigned)(p.a.n_requests * p.a.n_q), (unsigned)p.a.n_head), 64, 0, stream, p);
}

}  // extern "C"

// q4k_lora.hip -- q4k_lora_add (include/q4k_batch.h): low-rank adapters, one
// per token, beside a projection that all tokens share.
//
//   h[n][j]   = sum_k x[n][k] a[i][j][k]           (shrink), i = ids[n]
//   dst[n][m] = base[n][m] + scale[i] sum_j h[n][j] b[i][m][j]   (expand)
// h is F32 in the workspace: rank values a token.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "q4k_batch_host.h"
#include "q4k_device.h"

namespace q4k {

struct LoraParams {
    const char *a, *b;
    int64_t nb_a, nb_a_adapter, nb_b, nb_b_adapter, n_adapters;
    const float *scale;
    const int32_t *ranks;
    const char *x, *base;
    char *dst;
    int64_t nb_x, nb_base, nb_dst;
    const int32_t *ids;
    float *h;
    int64_t K, M, N;
    int rank;
};

__device__ __forceinline__ int adapter_rank(const LoraParams &p, int64_t i) {
    const int r = p.ranks ? p.ranks[i] : p.rank;
    return r < 0 ? 0 : r > p.rank ? p.rank : r;
}

template <class T>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraParams p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n = blockIdx.x;
    const int64_t i = p.ids[n];
    if (i < 0 || i >= p.n_adapters) return;
    const int r = adapter_rank(p, i);
    const float *x = reinterpret_cast<const float *>(p.x + n * p.nb_x);
    for (int j = wave; j < r; j += 4) {
        const T *a = reinterpret_cast<const T *>(p.a + i * p.nb_a_adapter + j * p.nb_a);
        float s = 0.0f;
        for (int64_t k = lane; k < p.K; k += 64) s += x[k] * (float)a[k];
        s = wave_sum(s);
        if (lane == 63) p.h[n * p.rank + j] = s;
    }
}

template <class T>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraParams p) {
    const int64_t n = blockIdx.y, m = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (m >= p.M) return;
    const int64_t i = p.ids[n];
    float y = p.base ? reinterpret_cast<const float *>(p.base + n * p.nb_base)[m] : 0.0f;
    if (i >= 0 && i < p.n_adapters) {
        const int r = adapter_rank(p, i);
        const T *b = reinterpret_cast<const T *>(p.b + i * p.nb_b_adapter + m * p.nb_b);
        float s = 0.0f;
        for (int j = 0; j < r; ++j) s += p.h[n * p.rank + j] * (float)b[j];
        y += (p.scale ? p.scale[i] : 1.0f) * s;
    }
    reinterpret_cast<float *>(p.dst + n * p.nb_dst)[m] = y;
}

static bool lora_sizes_ok(const q4k_lora *l, int64_t ne00, int64_t ne01, int64_t ne11) {
    return l && (l->type == Q4K_GGML_TYPE_F16 || l->type == Q4K_GGML_TYPE_BF16) && l->rank >= 1 &&
           l->rank <= Q4K_LORA_MAX_RANK && l->n_adapters >= 0 && l->n_adapters <= INT32_MAX && ne00 >= 0 && ne01 >= 0 &&
           ne11 >= 0 && ne00 <= INT32_MAX && ne01 <= INT32_MAX && ne11 <= INT32_MAX;
}

}  // namespace q4k

using namespace q4k;

extern "C" {

size_t q4k_lora_workspace_bytes(const q4k_lora *lora, int64_t ne00, int64_t ne01, int64_t ne11) {
    if (!lora_sizes_ok(lora, ne00, ne01, ne11)) return 0;
    return (size_t)ne11 * lora->rank * 4;
}

int q4k_lora_add(const q4k_lora *lora, int64_t ne00, int64_t ne01, const float *src1, int64_t ne11, int64_t nb11,
                 const int32_t *ids, const float *src2, int64_t nb21, float *dst, int64_t nb1, void *workspace,
                 size_t workspace_bytes, void *stream) {
    if (!lora_sizes_ok(lora, ne00, ne01, ne11)) return Q4K_EINVAL;
    const q4k_lora &l = *lora;
    if (!aligned(src1, 4) || !aligned(src2, 4) || !aligned(dst, 4) || !aligned(ids, 4) || !aligned(l.a, 2) ||
        !aligned(l.b, 2) || !aligned(l.scale, 4) || !aligned(l.ranks, 4))
        return Q4K_EINVAL;
    if (ne01 == 0 || ne11 == 0) return Q4K_OK;
    if (!dst || !ids || (ne00 > 0 && !src1)) return Q4K_EINVAL;
    if (nb11 % 4 != 0 || nb21 % 4 != 0 || nb1 % 4 != 0) return Q4K_EINVAL;
    if (ne11 > 1 && (nb11 < 4 * ne00 || nb1 < 4 * ne01 || (src2 && nb21 < 4 * ne01))) return Q4K_EINVAL;
    if (ne11 > 1 && src2 == dst && nb21 != nb1) return Q4K_EINVAL;
    if (l.n_adapters > 0) {
        if (!l.a || !l.b) return Q4K_EINVAL;
        if (l.nb_a % 2 != 0 || l.nb_b % 2 != 0 || l.nb_a_adapter % 2 != 0 || l.nb_b_adapter % 2 != 0) return Q4K_EINVAL;
        if (l.nb_a < 2 * ne00 || l.nb_b < 2 * l.rank || l.nb_a_adapter < 0 || l.nb_b_adapter < 0) return Q4K_EINVAL;
    }
    DeviceInfo *di;
    int st = device_info(&di);
    if (st != Q4K_OK) return st;
    if (ne11 > 65535) return Q4K_EUNSUPPORTED;
    Workspace ws;
    st = ws.begin(workspace, workspace_bytes, q4k_lora_workspace_bytes(lora, ne00, ne01, ne11), stream);
    if (st != Q4K_OK) return st;
    LoraParams p{};
    p.a = (const char *)l.a; p.b = (const char *)l.b;
    p.nb_a = l.nb_a; p.nb_a_adapter = l.nb_a_adapter; p.nb_b = l.nb_b; p.nb_b_adapter = l.nb_b_adapter;
    p.n_adapters = l.n_adapters; p.scale = l.scale; p.ranks = l.ranks;
    p.x = (const char *)src1; p.base = (const char *)src2; p.dst = (char *)dst;
    p.nb_x = nb11; p.nb_base = nb21; p.nb_dst = nb1;
    p.ids = ids; p.h = (float *)ws.ptr; p.K = ne00; p.M = ne01; p.N = ne11; p.rank = l.rank;
    const bool f16 = l.type == Q4K_GGML_TYPE_F16;
    st = launch(f16 ? lora_shrink_kernel<_Float16> : lora_shrink_kernel<__hip_bfloat16>, dim3((unsigned)ne11), 256, 0,
                stream, p);
    if (st == Q4K_OK)
        st = launch(f16 ? lora_expand_kernel<_Float16> : lora_expand_kernel<__hip_bfloat16>,
                    dim3((unsigned)((ne01 + 255) / 256), (unsigned)ne11), 256, 0, stream, p);
    return ws.end(st, stream);
}

}  // extern "C"

// q4k_logits.hip -- q4k_logits_adjust (include/q4k_batch.h): penalties for
// repeated tokens, biases and grammar masks on rows of logits.
//
// With c the number of times a token occurs in the row's history:
//   l = c > 0 ? (l > 0 ? l / repeat : l * repeat) : l
//   l = l - c * frequency - (c > 0 ? presence : 0)
//   l = l + bias (the last entry of the token), -inf where the mask bit is 0
// One pass over the logits: 8 bytes a logit, the bound.
#include <hip/hip_runtime.h>

#include "../../include/q4k_batch.h"
#include "q4k_batch_host.h"

namespace q4k {

struct LogitsParams {
    const char *src;
    char *dst;
    int64_t nb_src, nb_dst;
    int64_t n_vocab;
    int slices;
    q4k_logits_rules r;
};

constexpr int kLogitsThreads = 256, kLogitsPer = 8, kLogitsSlice = kLogitsThreads * kLogitsPer;

// [start[i], start[i+1]) clamped to [0, n): empty where the entries run backwards
__device__ __forceinline__ void list_range(const int64_t *start, int64_t i, int64_t n, int64_t &beg, int64_t &end) {
    beg = start[i];
    end = start[i + 1];
    if (beg < 0) beg = 0;
    if (end > n) end = n;
}

// One workgroup per slice of kLogitsSlice tokens of a row.  The slice's
// occurrences are counted in LDS with integer atomics, whose order does not
// change the counts; the same words then take the last bias entry of each token
// (the maximum of their numbers).
__global__ __launch_bounds__(kLogitsThreads) void logits_kernel(LogitsParams p) {
    __shared__ uint32_t cnt[kLogitsSlice];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x / p.slices;
    const int64_t v0 = (int64_t)(blockIdx.x % p.slices) * kLogitsSlice;
    const float *src = reinterpret_cast<const float *>(p.src + row * p.nb_src);
    float *dst = reinterpret_cast<float *>(p.dst + row * p.nb_dst);
    float l[kLogitsPer];
#pragma unroll
    for (int k = 0; k < kLogitsPer; ++k) {
        const int64_t v = v0 + k * kLogitsThreads + tid;
        l[k] = v < p.n_vocab ? src[v] : 0.0f;
    }
    const int lim = (int)(p.n_vocab - v0 < kLogitsSlice ? p.n_vocab - v0 : kLogitsSlice);
    int64_t beg = 0, end = 0;
    if (p.r.history) list_range(p.r.history_start, row, p.r.n_history, beg, end);
    if (beg < end) {
#pragma unroll
        for (int k = 0; k < kLogitsPer; ++k) cnt[k * kLogitsThreads + tid] = 0;
        __syncthreads();
        for (int64_t j = beg + tid; j < end; j += kLogitsThreads) {
            const int64_t t = (int64_t)p.r.history[j] - v0;
            if (t >= 0 && t < lim) atomicAdd(&cnt[t], 1u);
        }
        __syncthreads();
        const float rep = p.r.repeat ? p.r.repeat[row] : 1.0f;
        const float freq = p.r.frequency ? p.r.frequency[row] : 0.0f;
        const float pres = p.r.presence ? p.r.presence[row] : 0.0f;
#pragma unroll
        for (int k = 0; k < kLogitsPer; ++k) {
            const uint32_t c = cnt[k * kLogitsThreads + tid];
            if (c) {
                const float x = l[k] > 0.0f ? l[k] / rep : l[k] * rep;
                l[k] = x - (float)c * freq - pres;
            }
        }
    }
    int64_t bbeg = 0, bend = 0;
    if (p.r.bias_ids) list_range(p.r.bias_start, row, p.r.n_bias, bbeg, bend);
    if (bbeg < bend) {
        // own words only were read since the last barrier
#pragma unroll
        for (int k = 0; k < kLogitsPer; ++k) cnt[k * kLogitsThreads + tid] = 0;
        __syncthreads();
        for (int64_t j = bbeg + tid; j < bend; j += kLogitsThreads) {
            const int64_t t = (int64_t)p.r.bias_ids[j] - v0;
            if (t >= 0 && t < lim) atomicMax(&cnt[t], (uint32_t)(j - bbeg) + 1u);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kLogitsPer; ++k) {
            const uint32_t c = cnt[k * kLogitsThreads + tid];
            if (c) l[k] += p.r.bias[bbeg + c - 1];
        }
    }
    const uint32_t *mask = nullptr;
    if (p.r.mask) {
        const int64_t m = p.r.mask_rows ? p.r.mask_rows[row] : row;
        if (m >= 0 && m < p.r.n_masks)
            mask = reinterpret_cast<const uint32_t *>(reinterpret_cast<const char *>(p.r.mask) + m * p.r.nb_mask);
    }
#pragma unroll
    for (int k = 0; k < kLogitsPer; ++k) {
        const int64_t v = v0 + k * kLogitsThreads + tid;
        if (v < p.n_vocab) {
            if (mask && !((mask[v >> 5] >> (v & 31)) & 1u)) l[k] = -__builtin_inff();
            dst[v] = l[k];
        }
    }
}

}  // namespace q4k

using namespace q4k;

extern "C" int q4k_logits_adjust(const float *src, int64_t n_vocab, int64_t n_rows, int64_t nb_src,
                                 const q4k_logits_rules *rules, float *dst, int64_t nb_dst, void *stream) {
    if (!rules || n_vocab < 0 || n_rows < 0) return Q4K_EINVAL;
    const q4k_logits_rules &r = *rules;
    if (r.n_history < 0 || r.n_bias < 0 || r.n_masks < 0) return Q4K_EINVAL;
    if ((r.history != nullptr) != (r.history_start != nullptr)) return Q4K_EINVAL;
    if ((r.bias_ids != nullptr) != (r.bias != nullptr) || (r.bias_ids != nullptr) != (r.bias_start != nullptr))
        return Q4K_EINVAL;
    if (!aligned(src, 4) || !aligned(dst, 4) || !aligned(r.repeat, 4) || !aligned(r.frequency, 4) ||
        !aligned(r.presence, 4) || !aligned(r.history, 4) || !aligned(r.history_start, 8) ||
        !aligned(r.bias_ids, 4) || !aligned(r.bias, 4) || !aligned(r.bias_start, 8) || !aligned(r.mask, 4) ||
        !aligned(r.mask_rows, 4))
        return Q4K_EINVAL;
    if (n_vocab == 0 || n_rows == 0) return Q4K_OK;
    if (!src || !dst || n_vocab > INT32_MAX) return Q4K_EINVAL;
    if (nb_src % 4 != 0 || nb_dst % 4 != 0 || (n_rows > 1 && (nb_src < 4 * n_vocab || nb_dst < 4 * n_vocab)))
        return Q4K_EINVAL;
    if (src == dst && n_rows > 1 && nb_src != nb_dst) return Q4K_EINVAL;
    if (r.n_bias >= (int64_t)UINT32_MAX) return Q4K_EUNSUPPORTED;
    if (r.mask) {
        if (r.nb_mask % 4 != 0 || (r.n_masks > 1 && r.nb_mask < (n_vocab + 31) / 32 * 4)) return Q4K_EINVAL;
        if (!r.mask_rows && r.n_masks < n_rows) return Q4K_EINVAL;
    } else if (r.mask_rows) {
        return Q4K_EINVAL;
    }
    DeviceInfo *di;
    const int st = device_info(&di);
    if (st != Q4K_OK) return st;
    const int64_t slices = (n_vocab + kLogitsSlice - 1) / kLogitsSlice;
    if (n_rows > INT32_MAX / slices) return Q4K_EUNSUPPORTED;
    const LogitsParams p{reinterpret_cast<const char *>(src), reinterpret_cast<char *>(dst), nb_src, nb_dst, n_vocab,
                         (int)slices, r};
    return launch(logits_kernel, dim3((unsigned)(n_rows * slices)), kLogitsThreads, 0, stream, p);
}

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
#include "q4k_device.h"

namespace q4k {

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct LogitsParams {
    const char *src;
    char *dst;
    int64_t nb_src, nb_dst;
    int64_t n_vocab, n_rows;
    int slices;
    q4k_logits_rules r;
};

constexpr int kLogitsPer = 8;  // logits per thread, two 16-byte accesses

// [start[i], start[i+1]) clamped to [0, n): empty where the entries run backwards
__device__ __forceinline__ void list_range(const int64_t *start, int64_t i, int64_t n, int64_t &beg, int64_t &end) {
    beg = start[i];
    end = start[i + 1];
    if (beg < 0) beg = 0;
    if (end > n) end = n;
}

// f(entry, its number from beg) for the entries [beg, end) of a list, in 16-byte
// loads where they are aligned
template <int THREADS, class F>
__device__ __forceinline__ void for_list(const int32_t *list, int64_t beg, int64_t end, int tid, F f) {
    const int32_t *p = list + beg;
    const int64_t n = end - beg;
    int64_t head = (4 - (((uintptr_t)p >> 2) & 3)) & 3;
    if (head > n) head = n;
    const int64_t quads = (n - head) / 4;
    for (int64_t q = tid; q < quads; q += THREADS) {
        const int4 v = *reinterpret_cast<const int4 *>(p + head + 4 * q);
        const int64_t i = head + 4 * q;
        f(v.x, i);
        f(v.y, i + 1);
        f(v.z, i + 2);
        f(v.w, i + 3);
    }
    const int64_t tail = head + 4 * quads;
    if (tid < head) f(p[tid], tid);
    if (tid < n - tail) f(p[tail + tid], tail + tid);
}

// One workgroup per slice of THREADS * kLogitsPer tokens of a row; slices begin
// at 16-byte boundaries of the row of src, whatever its start.  The slice's
// occurrences are counted in LDS with integer atomics, and the last bias entry of
// each token is the maximum of their numbers: neither depends on the order.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void logits_kernel(LogitsParams p) {
    constexpr int SLICE = THREADS * kLogitsPer;
    __shared__ __attribute__((aligned(16))) uint32_t cnt[SLICE], last[SLICE];
    const int tid = threadIdx.x;
    // Workgroups go to the 8 XCDs in turn: a row's slices on one XCD read its
    // history through one L2.
    int64_t row, slice;
    if (p.n_rows >= 8) {
        const int64_t x = blockIdx.x & 7, i = blockIdx.x >> 3;
        row = i / p.slices * 8 + x;
        slice = i % p.slices;
        if (row >= p.n_rows) return;
    } else {
        row = blockIdx.x / p.slices;
        slice = blockIdx.x % p.slices;
    }
    const float *src = reinterpret_cast<const float *>(p.src + row * p.nb_src);
    float *dst = reinterpret_cast<float *>(p.dst + row * p.nb_dst);
    const int off = ((uintptr_t)src >> 2) & 3;
    const bool wide_out = (((uintptr_t)dst >> 2) & 3) == (uintptr_t)off;
    const int64_t v0 = slice * SLICE - off;  // of the slice's first place
    if (v0 >= p.n_vocab) return;
    f32x4 l[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int64_t v = v0 + (k * THREADS + tid) * 4;
        l[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (v >= 0 && v + 4 <= p.n_vocab) {
            l[k] = *reinterpret_cast<const f32x4 *>(src + v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (v + j >= 0 && v + j < p.n_vocab) l[k][j] = src[v + j];
        }
    }
    const uint32_t *mask = nullptr;
    if (p.r.mask) {
        const int64_t m = p.r.mask_rows ? p.r.mask_rows[row] : row;
        if (m >= 0 && m < p.r.n_masks)
            mask = reinterpret_cast<const uint32_t *>(reinterpret_cast<const char *>(p.r.mask) + m * p.r.nb_mask);
    }
    int64_t beg = 0, end = 0, bbeg = 0, bend = 0;
    if (p.r.history) list_range(p.r.history_start, row, p.r.n_history, beg, end);
    if (p.r.bias_ids) list_range(p.r.bias_start, row, p.r.n_bias, bbeg, bend);
    const bool has_h = beg < end, has_b = bbeg < bend;
    if (has_h || has_b) {
        const u32x4 z = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (has_h) *reinterpret_cast<u32x4 *>(cnt + (k * THREADS + tid) * 4) = z;
            if (has_b) *reinterpret_cast<u32x4 *>(last + (k * THREADS + tid) * 4) = z;
        }
        __syncthreads();
        // places of the slice that are tokens: [lo, hi)
        const int lo = v0 < 0 ? (int)-v0 : 0;
        const int hi = (int)(p.n_vocab - v0 < SLICE ? p.n_vocab - v0 : SLICE);
        const int base = (int)v0;
        auto place = [&](int32_t t) { return (int64_t)t - base >= lo && (int64_t)t - base < hi ? t - base : -1; };
        if (has_h)
            for_list<THREADS>(p.r.history, beg, end, tid, [&](int32_t t, int64_t) {
                const int at = place(t);
                if (at >= 0) atomicAdd(&cnt[at], 1u);
            });
        if (has_b)
            for_list<THREADS>(p.r.bias_ids, bbeg, bend, tid, [&](int32_t t, int64_t i) {
                const int at = place(t);
                if (at >= 0) atomicMax(&last[at], (uint32_t)i + 1u);
            });
        __syncthreads();
        if (has_h) {
            const float rep = p.r.repeat ? p.r.repeat[row] : 1.0f;
            const float freq = p.r.frequency ? p.r.frequency[row] : 0.0f;
            const float pres = p.r.presence ? p.r.presence[row] : 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const u32x4 c = *reinterpret_cast<const u32x4 *>(cnt + (k * THREADS + tid) * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c[j]) {
                        const float x = l[k][j] > 0.0f ? l[k][j] / rep : l[k][j] * rep;
                        l[k][j] = x - (float)c[j] * freq - pres;
                    }
            }
        }
        if (has_b) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const u32x4 c = *reinterpret_cast<const u32x4 *>(last + (k * THREADS + tid) * 4);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c[j]) l[k][j] += p.r.bias[bbeg + c[j] - 1];
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int64_t v = v0 + (k * THREADS + tid) * 4;
        if (mask) {
            // one word holds the four bits of a place that starts at a multiple of four
            const bool one = off == 0;
            uint32_t w = one && v < p.n_vocab ? mask[v >> 5] >> (v & 31) : 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (!one && v + j >= 0 && v + j < p.n_vocab) w = mask[(v + j) >> 5] >> ((v + j) & 31) << j;
                if (!((w >> j) & 1u)) l[k][j] = -__builtin_inff();
            }
        }
        if (wide_out && v >= 0 && v + 4 <= p.n_vocab) {
            *reinterpret_cast<f32x4 *>(dst + v) = l[k];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (v + j >= 0 && v + j < p.n_vocab) dst[v + j] = l[k][j];
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
    // Slices of 8192 logits where they fill the CUs: a row's history, which every
    // slice reads, is read the fewest times.  Else 2048, for more workgroups.
    const int64_t wide = (n_vocab + 3 + 8191) / 8192;
    const bool big = n_rows > di->cus / wide;
    const int64_t slices = big ? wide : (n_vocab + 3 + 2047) / 2048;
    const int64_t rows = n_rows >= 8 ? (n_rows + 7) / 8 * 8 : n_rows;
    if (rows > INT32_MAX / slices) return Q4K_EUNSUPPORTED;
    const LogitsParams p{reinterpret_cast<const char *>(src), reinterpret_cast<char *>(dst), nb_src, nb_dst, n_vocab,
                         n_rows, (int)slices, r};
    const dim3 grid((unsigned)(rows * slices));
    return big ? launch(logits_kernel<1024>, grid, 1024, 0, stream, p) : launch(logits_kernel<256>, grid, 256, 0, stream, p);
}

// q4k_logits.hip -- q4k_logits_adjust (include/q4k_batch.h): penalties for
// repeated tokens, biases and grammar masks on rows of logits.
//
// With c the number of times a token occurs in the row's history:
//   l = c > 0 ? (l > 0 ? l / repeat : l * repeat) : l
//   l = l - c * frequency - (c > 0 ? presence : 0)
//   l = l + bias (the last entry of the token), -inf where the mask bit is 0
// One pass over the logits: 8 bytes a logit and the history once per workgroup.
// 256 rows of 151936 logits with histories of 2048 to 8192 tokens take 73 us (4.3
// TB/s of what has to move; 61 us without histories, 5.2 TB/s; a copy reaches 5.4):
// memory bound, and with long histories bound by the counting in the slices of
// frequent tokens too.  Few rows are bound by the launch and three memory round
// trips (starts, histories, logits): 5.0 us for 32768 logits, 6.6 for 8 x 128256.
// (The form of 256 threads spills 16 bytes a lane at the 64 registers of eight waves a
// SIMD.)
#include <hip/hip_runtime.h>

#include "../../include/q4k_batch.h"
#include "q4k_batch.h"
#include "q4k_device.h"

namespace q4k {

struct LogitsParams {
    const char *src;
    char *dst;
    int64_t nb_src, nb_dst;
    int n_vocab, n_rows;
    int runs, run;  // workgroups of a row, slices of each
    q4k_logits_rules r;
};

constexpr int kLogitsPer = 8;  // logits per thread, two 16-byte accesses

// The list of row i: [start[i], start[i+1]) clamped to [0, n), empty where the
// entries run backwards.  Its length, and where it begins.  (Both ends are clamped
// before they are subtracted: starts may be any 64 bits.)
__device__ __forceinline__ int list_range(const int64_t *start, int64_t i, int64_t n, int64_t &beg) {
    beg = start[i];
    int64_t end = start[i + 1];
    beg = beg < 0 ? 0 : beg > n ? n : beg;
    end = end < beg ? beg : end > n ? n : end;
    end -= beg;
    return end > INT32_MAX - 8192 ? INT32_MAX - 8192 : (int)end;
}

// A list's entries in registers, H quads of them per thread of the workgroup:
// a row's history is read once for all its slices.  Entries that are not there
// are kNoToken, which no slice holds; those past THREADS * 4 * H are read when used.
constexpr int32_t kNoToken = INT32_MIN;
template <int THREADS, int H>
struct ListRegs {
    const int32_t *p;  // the first 16-byte aligned entry
    int quads;
    int4 v[H];
    int32_t edge;  // one of the entries before the first or after the last aligned quad

    __device__ __forceinline__ void load(const int32_t *list, int n, int tid) {
        int head = (4 - (int)(((uintptr_t)list >> 2) & 3)) & 3;
        if (head > n) head = n;
        quads = (n - head) / 4;
        p = list + head;
        const int tail = n - head - 4 * quads;  // at most three entries, as before the first quad
        edge = kNoToken;
        if (tid < head) edge = list[tid];
        else if (tid >= 4 && tid - 4 < tail) edge = p[4 * (int64_t)quads + tid - 4];
#pragma unroll
        for (int i = 0; i < H; ++i) {
            v[i] = make_int4(kNoToken, kNoToken, kNoToken, kNoToken);
            const int q = tid + i * THREADS;
            if (q < quads) v[i] = *reinterpret_cast<const int4 *>(p + 4 * (int64_t)q);
        }
    }
    template <class F>
    __device__ __forceinline__ void each(int tid, F f) const {
        auto quad = [&](const int4 &q) {
            f(q.x);
            f(q.y);
            f(q.z);
            f(q.w);
        };
#pragma unroll
        for (int i = 0; i < H; ++i)
            if (i * THREADS < quads) quad(v[i]);
        for (int q = H * THREADS + tid; q < quads; q += THREADS) quad(*reinterpret_cast<const int4 *>(p + 4 * (int64_t)q));
        f(edge);
    }
};

// A workgroup takes `run` slices of THREADS * kLogitsPer tokens of a row, one
// after the other, the next one's logits on their way while the lists are counted;
// slices begin at 16-byte boundaries of the row of src, whatever its start.  The
// slice's occurrences are counted in LDS with integer atomics, and the last bias
// entry of each token is the maximum of their numbers: neither depends on the order.
template <int THREADS, int H, bool NT>
__global__ __launch_bounds__(THREADS, 8) void logits_kernel(LogitsParams p) {
    constexpr int SLICE = THREADS * kLogitsPer;
    __shared__ __attribute__((aligned(16))) uint32_t cnt[SLICE], last[SLICE];
    const int tid = threadIdx.x;
    // Workgroups go to the 8 XCDs in turn: a row's workgroups on one XCD read its
    // history through one L2.
    int row, run0;
    if (p.n_rows >= 8) {
        const int i = blockIdx.x >> 3;
        row = i / p.runs * 8 + (blockIdx.x & 7);
        run0 = i % p.runs;
        if (row >= p.n_rows) return;
    } else {
        row = blockIdx.x / p.runs;
        run0 = blockIdx.x % p.runs;
    }
    const float *src = reinterpret_cast<const float *>(p.src + row * p.nb_src);
    float *dst = reinterpret_cast<float *>(p.dst + row * p.nb_dst);
    const int off = ((uintptr_t)src >> 2) & 3;
    const bool wide_out = (((uintptr_t)dst >> 2) & 3) == (uintptr_t)off;
    const uint32_t *mask = nullptr;
    if (p.r.mask) {
        const int64_t m = p.r.mask_rows ? p.r.mask_rows[row] : row;
        if (m >= 0 && m < p.r.n_masks)
            mask = reinterpret_cast<const uint32_t *>(reinterpret_cast<const char *>(p.r.mask) + m * p.r.nb_mask);
    }
    const int V = p.n_vocab;
    int v0 = run0 * p.run * SLICE - off;  // of the slice's first place
    if (v0 >= V) return;
    const int v1 = V - v0 > p.run * SLICE ? v0 + p.run * SLICE : V;

    // a slice's logits, and with masks the words of their bits (one word holds the
    // four of a place that starts at a multiple of four)
    f32x4 l[2], ln[2];
    uint32_t w[2], wn[2];
    auto load = [&](int s0, f32x4 (&x)[2], uint32_t (&m)[2]) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int v = s0 + (k * THREADS + tid) * 4;
            x[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            m[k] = 0;
            if (v >= 0 && v + 4 <= V) {
                x[k] = load4<NT>(src + v);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (v + j >= 0 && v + j < V) x[k][j] = src[v + j];
            }
            if (mask && off == 0 && v < V) m[k] = mask[v >> 5] >> (v & 31);
        }
    };
    load(v0, l, w);
    int64_t hbeg = 0, bbeg = 0;
    const int nh = p.r.history ? list_range(p.r.history_start, row, p.r.n_history, hbeg) : 0;
    const int nb = p.r.bias_ids ? list_range(p.r.bias_start, row, p.r.n_bias, bbeg) : 0;
    ListRegs<THREADS, H> hist;
    int32_t btok = kNoToken;  // bias entry tid
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    const u32x4 zero = {0, 0, 0, 0};
    if (nh) {
        hist.load(p.r.history + hbeg, nh, tid);
        if (p.r.repeat) rep = p.r.repeat[row];
        if (p.r.frequency) freq = p.r.frequency[row];
        if (p.r.presence) pres = p.r.presence[row];
    }
    if (tid < nb) btok = p.r.bias_ids[bbeg + tid];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (nh) *reinterpret_cast<u32x4 *>(cnt + (k * THREADS + tid) * 4) = zero;
        if (nb) *reinterpret_cast<u32x4 *>(last + (k * THREADS + tid) * 4) = zero;
    }

    for (; v0 < v1; v0 += SLICE) {
        if (v1 - v0 > SLICE) load(v0 + SLICE, ln, wn);
        if (nh || nb) {
            __syncthreads();  // the words are zero again
            // (places before token 0 or past the last one count too, and are not stored)
            if (nh)
                hist.each(tid, [&](int32_t t) {
                    const uint32_t at = (uint32_t)t - (uint32_t)v0;
                    if (at < (uint32_t)SLICE) atomicAdd(&cnt[at], 1u);
                });
            if (nb) {
                uint32_t at = (uint32_t)btok - (uint32_t)v0;
                if (at < (uint32_t)SLICE) atomicMax(&last[at], (uint32_t)tid + 1u);
                for (int i = THREADS + tid; i < nb; i += THREADS) {
                    at = (uint32_t)p.r.bias_ids[bbeg + i] - (uint32_t)v0;
                    if (at < (uint32_t)SLICE) atomicMax(&last[at], (uint32_t)i + 1u);
                }
            }
            __syncthreads();
            if (nh) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    u32x4 *at = reinterpret_cast<u32x4 *>(cnt + (k * THREADS + tid) * 4);
                    const u32x4 c = *at;
                    if (c[0] | c[1] | c[2] | c[3]) {
                        *at = zero;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float x = l[k][j] > 0.0f ? l[k][j] / rep : l[k][j] * rep;
                            if (c[j]) l[k][j] = x - (float)c[j] * freq - pres;
                        }
                    }
                }
            }
            if (nb) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    u32x4 *at = reinterpret_cast<u32x4 *>(last + (k * THREADS + tid) * 4);
                    const u32x4 c = *at;
                    if (c[0] | c[1] | c[2] | c[3]) {
                        *at = zero;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (c[j]) l[k][j] += p.r.bias[bbeg + c[j] - 1];
                    }
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int v = v0 + (k * THREADS + tid) * 4;
            if (mask) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t bit = w[k] >> j;
                    if (off != 0 && v + j >= 0 && v + j < V) bit = mask[(v + j) >> 5] >> ((v + j) & 31);
                    if (!(bit & 1u)) l[k][j] = -__builtin_inff();
                }
            }
            if (wide_out && v >= 0 && v + 4 <= V) {
                store4<NT>(dst + v, l[k]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (v + j >= 0 && v + j < V) dst[v + j] = l[k][j];
            }
            l[k] = ln[k];
            w[k] = wn[k];
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
    if (!src || !dst || n_vocab > INT32_MAX || n_rows > INT32_MAX) return Q4K_EINVAL;
    if (nb_src % 4 != 0 || nb_dst % 4 != 0 || (n_rows > 1 && (nb_src < 4 * n_vocab || nb_dst < 4 * n_vocab)))
        return Q4K_EINVAL;
    if (src == dst && n_rows > 1 && nb_src != nb_dst) return Q4K_EINVAL;
    if (n_vocab > (1 << 30)) return Q4K_EUNSUPPORTED;
    if (r.mask) {
        if (r.nb_mask % 4 != 0 || (r.n_masks > 1 && r.nb_mask < (n_vocab + 31) / 32 * 4)) return Q4K_EINVAL;
        if (!r.mask_rows && r.n_masks < n_rows) return Q4K_EINVAL;
    } else if (r.mask_rows) {
        return Q4K_EINVAL;
    }
    DeviceInfo *di;
    const int st = device_info(&di);
    if (st != Q4K_OK) return st;
    // Workgroups of 1024 threads where their slices of 8192 logits fill the CUs, four
    // a CU in all (two at a time; 256 rows of 151936 logits without histories 60.6 us
    // against 62.8 with two in all); else of 256 threads and 2048 logits, for more of
    // them.
    const int64_t wide = (n_vocab + 3 + 8191) / 8192;
    const bool big = n_rows > di->cus / wide;
    const int64_t slices = big ? wide : (n_vocab + 3 + 2047) / 2048;
    const int64_t per_row = 4 * (int64_t)di->cus / n_rows;
    const int64_t run = !big ? 1 : per_row < 1 ? slices : (slices + per_row - 1) / per_row;
    const int64_t runs = (slices + run - 1) / run;
    const int64_t rows = n_rows >= 8 ? (n_rows + 7) / 8 * 8 : n_rows;
    if (rows > INT32_MAX / runs) return Q4K_EUNSUPPORTED;
    const LogitsParams p{reinterpret_cast<const char *>(src), reinterpret_cast<char *>(dst), nb_src, nb_dst, (int)n_vocab,
                         (int)n_rows, (int)runs, (int)run, r};
    const dim3 grid((unsigned)(rows * runs));
    return !big                                ? launch(logits_kernel<256, 4, false>, grid, 256, 0, stream, p)
           : n_rows * n_vocab < kStreamFloats ? launch(logits_kernel<1024, 2, false>, grid, 1024, 0, stream, p)
                                               : launch(logits_kernel<1024, 2, true>, grid, 1024, 0, stream, p);
}

// q4k_sample.hip -- q4k_sample (include/q4k_step.h): the next token of each row of
// logits by temperature, top-k, top-p, min-p and a given random number.
//
// With a = log2(e) / temperature a token weighs w = 2^(a l), up to a factor of the
// row.  Cuts keep what is not below one token, in the order of falling logits and
// rising numbers, so they come from sums over a histogram of the exponents and an
// order within one of its bins:
//   1. one pass over the row counts tokens and sums their w in bins of 2^(1/32)
//   2. top-k, then top-p: the bin of the last token that is kept, and that token, from
//      the bin's tokens put in order (a bin of more than kList is divided again by
//      the logits' bits; equal logits are told apart by a count)
//   3. the kept w of each chunk of the row, the chunk that the random number falls
//      into, the token in it
// Sums of bins are integers (any order gives the same), all others are 64-bit floats
// in an order of their own: equal calls give equal bits.  A chunk whose largest
// logit is below the cut is not read again.
#include <hip/hip_runtime.h>

#include "../../include/q4k_step.h"
#include "q4k_batch.h"
#include "q4k_device.h"

namespace q4k {

struct SampleParams {
    const char *src;
    int64_t nb_src;
    int n_vocab, n_rows;
    int chunk, chunks;  // tokens of a chunk (a multiple of 256), chunks of a row
    int mass_bits;      // of a token's integer weight in its bin
    q4k_sample_rules r;
    int32_t *tokens;
    float *logprob;
};

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr int kBins = 4096, kOctave = 32;  // bins of the histogram, of a factor of two
constexpr int kAnchor = kBins - 1;         // the bin of the largest logit; what is below the last bin, 2^-128 of it, is never drawn
constexpr int kChunks = 1024, kList = 1024;

struct SampleLds {
    unsigned long long mass[kBins];
    uint32_t cnt[kBins];
    float cmax[kChunks];
    double cmass[kChunks];
    float list_l[kList], sort_l[kList];
    int list_i[kList], sort_i[kList];
    double scan[kSampleWaves];
    double scan2[kSampleWaves];
    int n_list, best;
    int found_i;
    double base_cnt, base_mass;
    float found_l;
};

__device__ __forceinline__ double shfl_up(double x, int d) {
    const unsigned long long b = __double_as_longlong(x);
    const uint32_t lo = __shfl_up((uint32_t)b, d), hi = __shfl_up((uint32_t)(b >> 32), d);
    return __longlong_as_double(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double shfl_xor(double x, int d) {
    const unsigned long long b = __double_as_longlong(x);
    const uint32_t lo = __shfl_xor((uint32_t)b, d), hi = __shfl_xor((uint32_t)(b >> 32), d);
    return __longlong_as_double(((unsigned long long)hi << 32) | lo);
}
__device__ __forceinline__ double wave_scan(double x) {  // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double y = shfl_up(x, d);
        if (lane >= d) x += y;
    }
    return x;
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) x += shfl_xor(x, d);
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}

// What is below x over the workgroup's threads in order, and the whole sum.
__device__ __forceinline__ double block_scan(double x, double *scan, double &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double inc = wave_scan(x);
    __syncthreads();
    if (lane == 63) scan[wave] = inc;
    __syncthreads();
    double before = 0.0;
    total = 0.0;
#pragma unroll
    for (int i = 0; i < kSampleWaves; ++i) {
        if (i < wave) before += scan[i];
        total += scan[i];
    }
    return before + (inc - x);
}

// A row's logits, and how they weigh.
struct SampleRow {
    const float *src;
    int n, chunk, chunks;
    float m;        // the largest logit
    bool flat;      // only logits equal to m count, all alike
    double a32;     // bins: a32 * (l - m) + kAnchor

    __device__ __forceinline__ float4 load(int i) const {
        float4 x;
        if (i + 4 <= n) {
            const f32x4 v = load4<false>(src + i);
            x = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            const float none = -__builtin_inff();
            x = make_float4(i < n ? src[i] : none, i + 1 < n ? src[i + 1] : none, i + 2 < n ? src[i + 2] : none, none);
        }
        x.x = clean(x.x);
        x.y = clean(x.y);
        x.z = clean(x.z);
        x.w = clean(x.w);
        return x;
    }
    // NaN is no candidate; zeros are equal whatever their sign
    __device__ __forceinline__ float clean(float l) const { return l != l ? -__builtin_inff() : l + 0.0f; }
    __device__ __forceinline__ bool counts(float l) const { return flat ? l == m : l > -__builtin_inff(); }
    __device__ __forceinline__ double place(float l) const { return flat ? kAnchor : __builtin_fma((double)l - (double)m, a32, kAnchor); }
    // the bin, below 0 where the token is none that counts
    __device__ __forceinline__ int bin(float l) const {
        if (!counts(l)) return -1;
        const double p = floor(place(l));
        return p < 0.0 ? -1 : (int)p;
    }
    // 2^(x / 32), x from place() less that of the largest
    __device__ __forceinline__ double weight(float l) const { return counts(l) ? exp2((place(l) - kAnchor) * (1.0 / kOctave)) : 0.0; }
    // in this order lower tokens of equal logits come first
    __device__ __forceinline__ static bool before(float l, int i, float k, int j) { return l > k || (l == k && i < j); }

    // f(token, four logits) of the chunks that on() asks for, each by one wave
    template <class ON, class F, class END>
    __device__ __forceinline__ void each(ON on, F f, END end) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        for (int c = wave; c < chunks; c += kSampleWaves) {
            if (!on(c)) continue;
            const int64_t c0 = (int64_t)c * chunk, c1 = c0 + chunk;
            for (int64_t i = c0; i < c1 && i < n; i += 256) f((int)i + lane * 4, load((int)i + lane * 4));
            end(c);
        }
    }
};

// ordered bits of a float: larger logits have larger keys
__device__ __forceinline__ uint32_t sample_key(float l) {
    const uint32_t b = __float_as_uint(l);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// 2^(x / 32) for 0 <= x < 1 in units of 1 / scale: the exponential's series (the next
// term is 2^-51 of it; exact at 0, where the largest logits are).
__device__ __forceinline__ unsigned long long sample_mass(double x, double scale) {
    const double y = x * (0.6931471805599453094 / kOctave);
    double e = 1.0 / 720.0;
    e = __builtin_fma(e, y, 1.0 / 120.0);
    e = __builtin_fma(e, y, 1.0 / 24.0);
    e = __builtin_fma(e, y, 1.0 / 6.0);
    e = __builtin_fma(e, y, 0.5);
    e = __builtin_fma(e, y, 1.0);
    e = __builtin_fma(e, y, 1.0);
    return (unsigned long long)(e * scale + 0.5);
}

__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleParams p) {
    extern __shared__ __attribute__((aligned(16))) char lds_bytes[];
    SampleLds &s = *reinterpret_cast<SampleLds *>(lds_bytes);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.x;
    const float inf = __builtin_inff();
    SampleRow x;
    x.src = reinterpret_cast<const float *>(p.src + row * p.nb_src);
    x.n = p.n_vocab;
    x.chunk = p.chunk;
    x.chunks = p.chunks;
    x.flat = false;
    x.a32 = 0.0;
    const float temperature = p.r.temperature ? p.r.temperature[row] : 1.0f;
    const float top_p = p.r.top_p ? p.r.top_p[row] : 1.0f;
    const float min_p = p.r.min_p ? p.r.min_p[row] : 0.0f;
    const int top_k = p.r.top_k ? p.r.top_k[row] : 0;
    float u = p.r.uniform ? p.r.uniform[row] : 0.0f;
    u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    const bool greedy = !p.r.uniform || !(temperature > 0.0f);
    const bool cut_k = top_k > 0 && top_k < p.n_vocab, cut_p = top_p < 1.0f;

    // the largest logit of each chunk and of the row, and its first token
    auto all = [](int) { return true; };
    float mc = -inf;
    x.each(all, [&](int, float4 l) { mc = fmaxf(fmaxf(fmaxf(mc, l.x), fmaxf(l.y, l.z)), l.w); },
           [&](int c) {
               mc = wave_max(mc);
               if (lane == 0) s.cmax[c] = mc;
               mc = -inf;
           });
    __syncthreads();
    x.m = wave_max(tid < p.chunks ? s.cmax[tid] : -inf);
    if (lane == 0) s.scan[wave] = x.m;
    if (tid == 0) s.found_i = INT32_MAX;
    __syncthreads();
    for (int i = 0; i < kSampleWaves; ++i) x.m = fmaxf(x.m, (float)s.scan[i]);
    if (x.m == -inf) {
        if (tid == 0) {
            p.tokens[row] = -1;
            if (p.logprob) p.logprob[row] = -inf;
        }
        return;
    }
    auto has_max = [&](int c) { return s.cmax[c] == x.m; };
    if (greedy) {
        int first = INT32_MAX;
        x.each(has_max, [&](int i, float4 l) {
            const int at = l.x == x.m ? i : l.y == x.m ? i + 1 : l.z == x.m ? i + 2 : l.w == x.m ? i + 3 : INT32_MAX;
            first = at < first ? at : first;
        }, [](int) {});
        if (first != INT32_MAX) atomicMin(&s.found_i, first);
        __syncthreads();
        if (tid == 0) {
            p.tokens[row] = s.found_i;
            if (p.logprob) p.logprob[row] = 0.0f;
        }
        return;
    }
    x.flat = x.m == inf;  // only the infinite ones count
    x.a32 = kOctave * 1.4426950408889634074 / (double)temperature;
    float last_l = -inf;  // the last token that is kept, in the order of the cuts
    int last_i = INT32_MAX;
    auto left_in = [&](float l, int i) { return !SampleRow::before(last_l, last_i, l, i); };
    if (cut_k || cut_p) {
        const double scale = (double)(1ull << p.mass_bits);
        // the histogram of what is left in
        auto count_all = [&]() {
            __syncthreads();
            for (int b = tid; b < kBins; b += kSampleThreads) {
                s.mass[b] = 0;
                s.cnt[b] = 0;
            }
            __syncthreads();
            x.each([&](int c) { return s.cmax[c] >= last_l; }, [&](int i, float4 l) {
                auto add = [&](float v, int t) {
                    if (!x.counts(v) || !left_in(v, t)) return;
                    const double at = x.place(v), f = floor(at);
                    if (f < 0.0) return;
                    atomicAdd(&s.mass[(int)f], sample_mass(at - f, scale));
                    atomicAdd(&s.cnt[(int)f], 1u);
                };
                add(l.x, i);
                add(l.y, i + 1);
                add(l.z, i + 2);
                add(l.w, i + 3);
            }, [](int) {});
            __syncthreads();
        };
        count_all();

        // The last token, in the order of the cuts, before which fewer than `most`
        // tokens (by_count) or less than `mass` lie; ahead: the sum of w up to it.
        auto find = [&](bool by_count, double most, double &ahead) {
            // thread t: bins 4095 - 4t and the three below it
            auto pick = [&](auto weight_of, int &bin, double &base_cnt, double &base_mass) {
                double cnt[4], mass[4], total;
                double sc = 0.0, sm = 0.0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int b = kBins - 1 - (tid * 4 + j);
                    cnt[j] = s.cnt[b];
                    mass[j] = cnt[j] != 0.0 ? weight_of(b) : 0.0;
                    sc += cnt[j];
                    sm += mass[j];
                }
                double bc = base_cnt + block_scan(sc, s.scan, total), bm = base_mass + block_scan(sm, s.scan2, total);
                if (tid == 0) s.best = -1;
                __syncthreads();
                int best = -1;
                double kc = 0.0, km = 0.0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (cnt[j] != 0.0 && ((by_count ? bc < most : bm < most) || bc == 0.0)) {
                        best = tid * 4 + j;
                        kc = bc;
                        km = bm;
                    }
                    bc += cnt[j];
                    bm += mass[j];
                }
                if (best >= 0) atomicMax(&s.best, best);
                __syncthreads();
                if (best >= 0 && s.best == best) {
                    s.base_cnt = kc;
                    s.base_mass = km;
                }
                __syncthreads();
                bin = kBins - 1 - s.best;
                base_cnt = s.base_cnt;
                base_mass = s.base_mass;
            };
            double base_cnt = 0.0, base_mass = 0.0;
            int bin;
            const double unit = 1.0 / scale;
            pick([&](int b) { return (double)s.mass[b] * unit * exp2((b - kAnchor) * (1.0 / kOctave)); }, bin, base_cnt, base_mass);
            uint32_t n = s.cnt[bin];
            const int bin0 = bin;
            // the keys of the bin's logits, divided until few are left or all are equal
            uint32_t lo = 0, hi = 0xffffffffu;
            auto in_bin = [&](float l, int i) { return x.bin(l) == bin0 && sample_key(l) >= lo && sample_key(l) <= hi && left_in(l, i); };
            auto maybe = [&](int c) { return x.bin(s.cmax[c]) >= bin0; };
            __syncthreads();
            while (n > kList && lo != hi) {
                // (the histogram of the bins is built again below, where it is needed again)
                const int shift = 32 - __builtin_clz((hi - lo) | 4095u) - 12;
                for (int b = tid; b < kBins; b += kSampleThreads) {
                    s.mass[b] = 0;
                    s.cnt[b] = 0;
                }
                __syncthreads();
                x.each(maybe, [&](int i, float4 l) {
                    auto add = [&](float v, int t) {
                        if (!in_bin(v, t)) return;
                        const double at = x.place(v);
                        atomicAdd(&s.mass[(sample_key(v) - lo) >> shift], sample_mass(at - floor(at), scale));
                        atomicAdd(&s.cnt[(sample_key(v) - lo) >> shift], 1u);
                    };
                    add(l.x, i);
                    add(l.y, i + 1);
                    add(l.z, i + 2);
                    add(l.w, i + 3);
                }, [](int) {});
                __syncthreads();
                const double w0 = unit * exp2((bin0 - kAnchor) * (1.0 / kOctave));
                pick([&](int b) { return (double)s.mass[b] * w0; }, bin, base_cnt, base_mass);
                n = s.cnt[bin];
                lo += (uint32_t)bin << shift;
                if (hi - lo > (1u << shift) - 1) hi = lo + ((1u << shift) - 1);
                __syncthreads();
            }
            if (n > kList) {
                // equal logits: how many of them, and the number of the last one
                const uint32_t b = lo & 0x80000000u ? lo ^ 0x80000000u : ~lo;
                const float l = __uint_as_float(b);
                const double w = x.weight(l);
                double keep = by_count ? most - base_cnt : ceil((most - base_mass) / w);
                keep = keep < 1.0 ? 1.0 : keep > n ? n : keep;
                int mine = 0;
                x.each(maybe, [&](int, float4 v) { mine += (v.x == l) + (v.y == l) + (v.z == l) + (v.w == l); },
                       [&](int c) {
                           const double sum = wave_sum((double)mine);
                           if (lane == 0) s.cmass[c] = sum;
                           mine = 0;
                       });
                __syncthreads();
                double total;
                const double have = tid < p.chunks && maybe(tid) ? s.cmass[tid] : 0.0;
                const double before = block_scan(have, s.scan, total);
                if (before < keep && before + have >= keep) {
                    s.best = tid;
                    s.base_cnt = keep - before;
                }
                __syncthreads();
                const int c = s.best;
                if (wave == 0) {
                    double left = s.base_cnt;
                    const int64_t c0 = (int64_t)c * x.chunk;
                    for (int64_t i = c0; i < c0 + x.chunk && i < x.n && left > 0.0; i += 256) {
                        const float4 v = x.load((int)i + lane * 4);
                        const int is[4] = {v.x == l, v.y == l, v.z == l, v.w == l};
                        const double all4 = is[0] + is[1] + is[2] + is[3], inc = wave_scan(all4);
                        double at = inc - all4;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            at += is[j];
                            if (is[j] && at == left) s.found_i = (int)i + lane * 4 + j;
                        }
                        left -= __shfl((float)inc, 63);
                    }
                }
                __syncthreads();
                last_l = l;
                last_i = s.found_i;
                ahead = base_mass + keep * w;
                __syncthreads();
                return bin0;
            }
            // the tokens of the bin in order
            if (tid == 0) s.n_list = 0;
            __syncthreads();
            x.each(maybe, [&](int i, float4 l) {
                auto add = [&](float v, int t) {
                    if (!in_bin(v, t)) return;
                    const int at = atomicAdd(&s.n_list, 1);
                    s.list_l[at] = v;
                    s.list_i[at] = t;
                };
                add(l.x, i);
                add(l.y, i + 1);
                add(l.z, i + 2);
                add(l.w, i + 3);
            }, [](int) {});
            __syncthreads();
            const int m = s.n_list;
            if (tid < m) {
                const float l = s.list_l[tid];
                const int t = s.list_i[tid];
                int rank = 0;
                for (int j = 0; j < m; ++j) rank += SampleRow::before(s.list_l[j], s.list_i[j], l, t);
                s.sort_l[rank] = l;
                s.sort_i[rank] = t;
            }
            __syncthreads();
            const double w = tid < m ? x.weight(s.sort_l[tid]) : 0.0;
            double total;
            const double at_mass = base_mass + block_scan(w, s.scan, total), at_cnt = base_cnt + tid;
            if (tid == 0) s.best = 0;
            __syncthreads();
            const bool kept = tid < m && ((by_count ? at_cnt < most : at_mass < most) || at_cnt == 0.0);
            if (kept) atomicMax(&s.best, tid);
            __syncthreads();
            if (tid == s.best) s.base_mass = at_mass + w;
            last_l = s.sort_l[s.best];
            last_i = s.sort_i[s.best];
            __syncthreads();
            ahead = s.base_mass;
            return bin0;
        };
        double ahead = 0.0;
        bool limited = false;
        if (cut_k) {
            find(true, (double)top_k, ahead);
            limited = true;
        }
        if (cut_p) {
            double whole = ahead;
            if (limited) {
                count_all();
            } else {
                double sm = 0.0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int b = kBins - 1 - (tid * 4 + j);
                    if (s.cnt[b]) sm += (double)s.mass[b] / scale * exp2((b - kAnchor) * (1.0 / kOctave));
                }
                block_scan(sm, s.scan, whole);
            }
            const float kl = last_l;
            const int ki = last_i;
            find(false, (double)top_p * whole, ahead);
            // (a rounding of the sums must not bring back what top-k cut off)
            if (limited && SampleRow::before(kl, ki, last_l, last_i)) {
                last_l = kl;
                last_i = ki;
            }
        }
    }
    // the kept w of each chunk
    const double min_w = min_p > 0.0f ? (double)fminf(min_p, 1.0f) : 0.0;
    auto kept_w = [&](float l, int i) {
        if (!x.counts(l) || !left_in(l, i)) return 0.0;
        const double w = x.weight(l);
        return w >= min_w ? w : 0.0;
    };
    auto kept_chunk = [&](int c) { return s.cmax[c] >= last_l && s.cmax[c] > -inf; };
    double sum = 0.0;
    __syncthreads();
    x.each(kept_chunk, [&](int i, float4 l) {
        sum += (kept_w(l.x, i) + kept_w(l.y, i + 1)) + (kept_w(l.z, i + 2) + kept_w(l.w, i + 3));
    }, [&](int c) {
        sum = wave_sum(sum);
        if (lane == 0) s.cmass[c] = sum;
        sum = 0.0;
    });
    __syncthreads();
    double total;
    const double have = tid < p.chunks && kept_chunk(tid) ? s.cmass[tid] : 0.0;
    const double before = block_scan(have, s.scan, total);
    const double target = (double)u * total;
    if (tid == 0) s.best = -1;
    __syncthreads();
    // the first chunk whose sum passes the target; where rounding leaves none, the last with any
    if (have > 0.0 && before <= target) atomicMax(&s.best, tid);
    __syncthreads();
    if (tid == s.best) s.base_mass = target - before;
    __syncthreads();
    if (wave == 0) {
        double left = s.base_mass;
        const int64_t c0 = (int64_t)(s.best < 0 ? 0 : s.best) * x.chunk;
        int token = -1;
        float logit = 0.0f;
        bool done = false;
        for (int64_t i = c0; i < c0 + x.chunk && i < x.n && !done; i += 256) {
            const int t = (int)i + lane * 4;
            const float4 l = x.load(t);
            const float v[4] = {l.x, l.y, l.z, l.w};
            double w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = kept_w(v[j], t + j);
            const double mine = (w[0] + w[1]) + (w[2] + w[3]), inc = wave_scan(mine);
            double at = inc - mine;
            int pick = -1, any = -1;
#pragma unroll
            for (int j = 3; j >= 0; --j) {
                double upto = at;
#pragma unroll
                for (int k = 0; k <= j; ++k) upto += w[k];
                if (w[j] > 0.0 && any < 0) any = j;
                if (w[j] > 0.0 && upto > left) pick = j;
            }
            const unsigned long long passed = __ballot(pick >= 0), some = __ballot(any >= 0);
            if (passed) {
                const int from = __builtin_ctzll(passed);
                const int j = __shfl(pick, from);
                token = (int)i + from * 4 + j;
                logit = __shfl(j == 0 ? v[0] : j == 1 ? v[1] : j == 2 ? v[2] : v[3], from);
                done = true;
            } else if (some) {  // (so far the last)
                const int from = 63 - __builtin_clzll(some);
                const int j = __shfl(any, from);
                token = (int)i + from * 4 + j;
                logit = __shfl(j == 0 ? v[0] : j == 1 ? v[1] : j == 2 ? v[2] : v[3], from);
            }
            left -= wave_sum(mine);
        }
        if (lane == 0) {
            p.tokens[row] = token;
            if (p.logprob) p.logprob[row] = (float)log(x.weight(logit) / total);
        }
    }
}

static bool sample_sizes(int64_t n_vocab, int64_t n_rows) { return n_vocab >= 0 && n_rows >= 0 && n_vocab <= INT32_MAX && n_rows <= INT32_MAX; }

}  // namespace q4k

using namespace q4k;

extern "C" {

size_t q4k_sample_workspace_bytes(int64_t n_vocab, int64_t n_rows) {
    (void)n_vocab;
    (void)n_rows;
    return 0;
}

int q4k_sample(const float *src, int64_t n_vocab, int64_t n_rows, int64_t nb_src, const q4k_sample_rules *rules, int32_t *tokens, float *logprob,
               void *workspace, size_t workspace_bytes, void *stream) {
    (void)workspace;
    (void)workspace_bytes;
    if (!rules || !sample_sizes(n_vocab, n_rows)) return Q4K_EINVAL;
    const q4k_sample_rules &r = *rules;
    if (!aligned(src, 4) || !aligned(r.temperature, 4) || !aligned(r.top_k, 4) || !aligned(r.top_p, 4) || !aligned(r.min_p, 4) ||
        !aligned(r.uniform, 4) || !aligned(tokens, 4) || !aligned(logprob, 4))
        return Q4K_EINVAL;
    if (n_rows == 0) return Q4K_OK;
    if ((!src && n_vocab > 0) || !tokens || nb_src % 4 != 0 || (n_rows > 1 && nb_src < 4 * n_vocab)) return Q4K_EINVAL;
    if (n_vocab > (1 << 30)) return Q4K_EUNSUPPORTED;
    DeviceInfo *di;
    int st = device_info(&di);
    if (st != Q4K_OK) return st;
    int chunk = 256, bits = 0;
    while ((n_vocab + chunk - 1) / chunk > kChunks) chunk *= 2;
    while ((int64_t)1 << bits < n_vocab) ++bits;
    const SampleParams p{reinterpret_cast<const char *>(src), nb_src, (int)n_vocab, (int)n_rows, chunk, (int)((n_vocab + chunk - 1) / chunk),
                         62 - bits < 44 ? 62 - bits : 44, r, tokens, logprob};
    st = ensure_lds(di, reinterpret_cast<const void *>(&sample_kernel), (int)sizeof(SampleLds));
    if (st != Q4K_OK) return st;
    return launch(sample_kernel, dim3((unsigned)n_rows), kSampleThreads, (int)sizeof(SampleLds), stream, p);
}

}  // extern "C"

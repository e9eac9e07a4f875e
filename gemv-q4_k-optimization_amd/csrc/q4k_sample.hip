// q4k_sample.hip -- q4k_sample (include/q4k_step.h): the next token of each row of
// logits by temperature, top-k, top-p, min-p and a given random number.
//
// With a = log2(e) / temperature a token weighs w = 2^(a l), up to a factor of the
// row.  Cuts keep what is not below one token, in the order of falling logits and
// rising numbers, so they come from sums over a histogram of the exponents and an
// order within one of its bins:
//   scan  parts of the rows, read once: the largest logit of each chunk of 256 and
//         what the row's rules need, counts and sums of w in bins of 2^(1/24), or
//         without cuts the sum of each chunk
//   draw  workgroups of all parts of the row find the bin of the last token that is kept
//         from the scan's octaves and then that octave's bins, each for itself, and read
//         the chunks that matter again: the tokens from that bin up where they are few
//         (kList), else the sums by chunks of what is above it and the bin's own tokens.
//         The last workgroup of a row cuts the list to the last token that is kept, sums it
//         by chunks, and finds the chunk that the random number falls into and the token
//         in it.  What does not fit this, one workgroup does from the row alone: rows out of the
//         scan's reach, top-k and top-p both past kList, a bin of more than kList tokens
//         (divided by the logits' bits until it has less or only equal ones, which are
//         told apart by a count).  The last is no rare case of top-p at raised temperatures:
//         of 151936 normal logits of deviation 2.5 the bin of 0.95 has 720 tokens at 1.2, 990 at
//         1.5 and 1220 at 2, and 256 such rows take 140 us at 1.2, 345 at 1.5 and 405 at 2, 8 rows of 262144 41 us at 1.0
//         and 540 to 590 from 1.2 on.
// (A CU reads some 13 bytes a cycle from beyond the L2s, so that one workgroup a row would
// take longer for a row's logits, or for whole histograms, than all else takes.)
// Sums of bins are integers (any order gives the same), all others are 64-bit floats
// in an order of their own: equal calls give equal bits.  A chunk whose largest
// logit is below the cut is not read again.
//
// Bound by: 256 rows of 151936 (156 MB) 55 us of scan, of which the reads alone take 30 and the
// 64-bit arithmetic as long, beside them in part; 76 us of draw, one workgroup a CU for its
// registers (two, at 128 of them, spill: 8 rows 35 us for both kernels instead of 33).
// Few rows: chains of round trips (1 x 32768: 6 + 17 us).  In three launches, with
// one that finds the bins alone: 174 us and 25.
#include <hip/hip_runtime.h>

#include "../../include/q4k_step.h"
#include "q4k_batch.h"
#include "q4k_device.h"
#include "q4k_scan.h"

// A token's weight is compared with the same token's, worked out elsewhere: products and
// sums are fused where fma() says so only.
#pragma clang fp contract(off)

namespace q4k {

constexpr int kDrawThreads = 512;
constexpr int kScanThreads = 512, kScanWaves = kScanThreads / 64, kTile = kScanThreads * 8;
constexpr int kOctave = 24, kOctaves = 64, kBins = kOctaves * kOctave;  // what is below the last bin is never drawn
constexpr int kMassBits = 44;  // of a token's integer weight in its bin (of up to 2^18, what a scan numbers)
constexpr int kChunk = 256, kChunks = 1024, kList = 1024, kShort = 256, kParts = 16;
// Rows whose a l is past this (in bins) lose bits of w and are not scanned: the pick
// takes them by the differences from their largest logit.
constexpr double kReach = 16384.0;
// Sums nearer to a border than this part of it count as equal to it.
constexpr double kNear = 0x1p-40;

// What a part of a row was found to hold.
struct SamplePart {
    double base;    // bin i is place base - kBins + i
    float skipped;  // the largest logit of tiles that were too low to be placed
    int used;       // whether some tile was not
    double octave_mass[kOctaves];  // of an octave's bins, in units of its lowest one
    uint32_t octave_cnt[kOctaves];
    unsigned long long mass[kBins];
    uint32_t cnt[kBins];
};

// What the workgroups of a row share: the list of tokens, and how many are done.
struct SampleList {
    int n, done;
    float l[kList];
    int i[kList];
};

struct SampleParams {
    const char *src;
    int64_t nb_src;
    int n_vocab, n_rows;
    int chunk, chunks;  // tokens of a chunk (a multiple of 256), chunks of a row
    int past_bits;      // sample_past's
    int parts, tiles;   // of a row (0: not scanned); of a part
    int shares;         // workgroups of a row's draw
    SamplePart *part;
    float *cmax;        // [rows][kChunks]
    double *cmass;
    SampleList *list;
    float *pad;         // [rows][4], of rows of fewer
    q4k_sample_rules r;
    int32_t *tokens;
    float *logprob;
};

// A row's rules.
struct SampleRules {
    float temperature, top_p, min_p;
    int top_k;
    float u;
    bool greedy, cut;
    __device__ __forceinline__ SampleRules(const SampleParams &p, int row) {
        temperature = p.r.temperature ? p.r.temperature[row] : 1.0f;
        top_p = p.r.top_p ? p.r.top_p[row] : 1.0f;
        min_p = p.r.min_p ? p.r.min_p[row] : 0.0f;
        top_k = p.r.top_k ? p.r.top_k[row] : 0;
        if (top_k < 0 || top_k >= p.n_vocab) top_k = 0;
        top_p = top_p < 1.0f ? fmaxf(top_p, 0.0f) : 1.0f;
        min_p = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;
        u = p.r.uniform ? p.r.uniform[row] : 0.0f;
        u = u > 0.0f ? fminf(u, 0.99999994f) : 0.0f;
        greedy = !p.r.uniform || !(temperature > 0.0f);
        cut = !greedy && (top_k > 0 || top_p < 1.0f);
    }
    // neither cuts nor a bound: every chunk's sum is what the draw needs
    __device__ __forceinline__ bool free() const { return !greedy && !cut && min_p == 0.0f; }
    // bins per unit of a logit
    __device__ __forceinline__ double rate() const { return kOctave * 1.4426950408889634074 / (double)temperature; }
};

// ---- sums and largest values over a wave's lanes ----
__device__ __forceinline__ double last_lane(double x) { return lane_of(x, 63); }
__device__ __forceinline__ double wave_sum(double x) { return last_lane(wave_scan(x)); }
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_max(float x) {
    const int b = __float_as_int(x);
    return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp(b, b, CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float x) {
    x = dpp_max<0x111, 0xf>(x);
    x = dpp_max<0x112, 0xf>(x);
    x = dpp_max<0x114, 0xf>(x);
    x = dpp_max<0x118, 0xf>(x);
    x = dpp_max<0x142, 0xa>(x);
    x = dpp_max<0x143, 0xc>(x);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// Two values' largest, four values' sums: halves and quarters of the wave take one each, the
// last lane of which ends up with its result.
typedef uint32_t lane_pair __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float wave_max2(float x, float y) {  // lanes 31 and 63
    const lane_pair h = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    x = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
    x = dpp_max<0x111, 0xf>(x);
    x = dpp_max<0x112, 0xf>(x);
    x = dpp_max<0x114, 0xf>(x);
    x = dpp_max<0x118, 0xf>(x);
    return dpp_max<0x142, 0xa>(x);
}
template <bool ROWS>
__device__ __forceinline__ double half_sums(double x, double y) {
    const unsigned long long a = __double_as_longlong(x), b = __double_as_longlong(y);
    lane_pair lo, hi;
    if (ROWS) {
        lo = __builtin_amdgcn_permlane16_swap((uint32_t)a, (uint32_t)b, false, false);
        hi = __builtin_amdgcn_permlane16_swap((uint32_t)(a >> 32), (uint32_t)(b >> 32), false, false);
    } else {
        lo = __builtin_amdgcn_permlane32_swap((uint32_t)a, (uint32_t)b, false, false);
        hi = __builtin_amdgcn_permlane32_swap((uint32_t)(a >> 32), (uint32_t)(b >> 32), false, false);
    }
    return __longlong_as_double(((unsigned long long)hi[0] << 32) | lo[0]) + __longlong_as_double(((unsigned long long)hi[1] << 32) | lo[1]);
}
__device__ __forceinline__ double row_sums(double x) {
    x += dpp64<0x111, 0xf>(x);
    x += dpp64<0x112, 0xf>(x);
    x += dpp64<0x114, 0xf>(x);
    return x + dpp64<0x118, 0xf>(x);
}
__device__ __forceinline__ double wave_sum2(double x, double y) {  // lanes 31 and 63
    x = row_sums(half_sums<false>(x, y));
    return x + dpp64<0x142, 0xa>(x);
}
__device__ __forceinline__ double wave_sum4(double a, double b, double c, double d) {  // lanes 15, 47, 31 and 63
    return row_sums(half_sums<true>(half_sums<false>(a, b), half_sums<false>(c, d)));
}

// Four logits of a row of n (4 or more) from token i, read from where the row has four (no
// branch between loads, so that all of a thread's are on their way together); sample_fix moves
// them to their places, past the row -inf.
__device__ __forceinline__ f32x4 sample_load(const float *src, int n, int i) { return load4<false>(src + (i < n - 4 ? i : n - 4)); }
__device__ __forceinline__ f32x4 sample_fix(f32x4 x, int n, int i) {
    const int by = i - (n - 4);
    if (by <= 0) return x;
    f32x4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        y[j] = -__builtin_inff();
#pragma unroll
        for (int k = j + 1; k < 4; ++k) y[j] = k - j == by ? x[k] : y[j];
    }
    return y;
}
// (zeros are equal whatever their sign)
__device__ __forceinline__ float sample_clean(float l) { return l != l ? -__builtin_inff() : l + 0.0f; }

// The whole number nearest to t (within 2^31 of 0), and what t is past it: 1.5 * 2^52 more
// leaves it in the last bits, two additions where floor and a conversion take 20 cycles.
__device__ __forceinline__ int sample_place(double t, double &past) {
    const double r = t + 0x1.8p52;
    past = t - (r - 0x1.8p52);
    return (int)(uint32_t)__double_as_longlong(r);
}
// scale * 2^(x / 24) + plus for |x| <= 1/2: the exponential's series (the next term is
// 2^-46 of it).
__device__ __forceinline__ double sample_exp(double x, double scale, double plus) {
    constexpr double k = 0.6931471805599453094 / kOctave;
    double e = k * k * k * k * k / 120.0;
    e = __builtin_fma(e, x, k * k * k * k / 24.0);
    e = __builtin_fma(e, x, k * k * k / 6.0);
    e = __builtin_fma(e, x, k * k / 2.0);
    e = __builtin_fma(e, x, k);
    return __builtin_fma(e * x, scale, scale + plus);
}
// 2^((b - kBins) / 24) times e near 1 (or any sum), from the 24 powers of an octave.
__device__ __forceinline__ double sample_weight(const double *octave, int b, double e) {
    const int q = b * 2731 >> 16;  // b / 24, rounded down, from -1 to 8192
    return __longlong_as_double(__double_as_longlong(octave[b - q * kOctave] * e) + ((long long)(q - kOctaves) << 52));
}
__device__ __forceinline__ double sample_weight_sum(const double *octave, int b, double sum) {
    const int q = b * 2731 >> 16;
    return ldexp(octave[b - q * kOctave] * sum, q - kOctaves);
}
// as an integer of bits and one more, scale 2^bits: 2^52 more leaves it in the last bits
__device__ __forceinline__ unsigned long long sample_mass(double x, double scale) {
    return __double_as_longlong(sample_exp(x, scale, 0x1p52)) & 0xfffffffffffffull;
}
// What it is past 1, within 2^-6.1 of it, as an integer with a sign: of 2^30 tokens it leaves room
// for 39 bits, where the whole weight would for 33.
__device__ __forceinline__ unsigned long long sample_past(double x, double scale) {
    return (unsigned long long)(__double_as_longlong(sample_exp(x, scale, 0x1.8p52 - scale)) - __double_as_longlong(0x1.8p52));
}

// ---- scan: parts of the rows ----
// Tiles of 4096 logits, eight a thread, the next one on its way.  The bins are a ring
// about the place of the largest logit so far, in whole octaves.
__global__ __launch_bounds__(kScanThreads) void sample_scan_kernel(SampleParams p) {
    __shared__ unsigned long long mass[kBins];
    __shared__ uint32_t cnt[kBins];
    __shared__ double octave[kOctave];  // the powers of 2^(1/24)
    __shared__ float tops[2][kScanWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.x / p.parts, part = blockIdx.x - row * p.parts;
    const float *src = reinterpret_cast<const float *>(p.src + row * p.nb_src);
    const int64_t beg = (int64_t)part * p.tiles * kTile;
    if (beg >= p.n_vocab) return;
    const int64_t end = beg + (int64_t)p.tiles * kTile;
    // thread: tokens wave * 512 + lane * 4 and 256 past it
    const int at = wave * 2 * kChunk + lane * 4;
    f32x4 next[2];
    next[0] = sample_load(src, p.n_vocab, (int)beg + at);
    next[1] = sample_load(src, p.n_vocab, (int)beg + at + kChunk);
    const SampleRules r(p, row);
    const bool cut = r.cut, by_mass = r.top_k == 0, free = r.free();  // (top-k needs counts alone)
    const double rate = r.rate(), scale = (double)(1ull << kMassBits);
    if (tid < kOctave) octave[tid] = exp2(tid * (1.0 / kOctave));
    if (part == 0 && tid == 0) p.list[row].n = p.list[row].done = 0;
    if (free) __syncthreads();
    float *cmax = p.cmax + (int64_t)row * kChunks;
    double *cmass = p.cmass + (int64_t)row * kChunks;
    double base = 0.0;  // bins: places base - kBins .. base - 1
    int off = 0;        // where bin 0 is in the ring
    bool used = false;
    float skipped = -__builtin_inff();
    int par = 0;
    for (int64_t t0 = beg; t0 < end && t0 < p.n_vocab; t0 += kTile, par ^= 1) {
        f32x4 l[2] = {next[0], next[1]};
        next[0] = sample_load(src, p.n_vocab, (int)t0 + kTile + at);  // (behind the part: what is not used)
        next[1] = sample_load(src, p.n_vocab, (int)t0 + kTile + at + kChunk);
        if (t0 + kTile > p.n_vocab) {
            l[0] = sample_fix(l[0], p.n_vocab, (int)t0 + at);
            l[1] = sample_fix(l[1], p.n_vocab, (int)t0 + at + kChunk);
        }
        float top[2];
        double sum[2] = {};
#pragma unroll
        for (int k = 0; k < 2; ++k) top[k] = fmaxf(fmaxf(l[k][0], l[k][1]), fmaxf(l[k][2], l[k][3]));  // (NaN passed over)
        const float both = wave_max2(top[0], top[1]);
        top[0] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(both), 31));
        top[1] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(both), 63));
        // lanes 31 and 63 write the first and the second chunk's
        const int c = (int)(t0 + at - lane * 4) / kChunk + (lane >> 5);
        const bool writes = (lane & 31) == 31 && c < p.chunks;
        if (writes) cmax[c] = sample_clean(both);
        if (free) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const double cb = __builtin_rint((double)top[k] * rate) + 1.0;
                if (!(fabs(cb) < kReach)) continue;
                const int low = (int)cb - kBins;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    double past;
                    const int i = sample_place(fmax((double)l[k][j] * rate, cb - (kBins + 1)), past) - low;
                    const double w = sample_weight(octave, i, sample_exp(past, 1.0, 0.0));
                    sum[k] += i >= 0 ? w : 0.0;
                }
            }
            const double sums = wave_sum2(sum[0], sum[1]);
            if (writes) cmass[c] = sums;
        }
        if (!cut) continue;
        if (lane == 0) tops[par][wave] = fmaxf(top[0], top[1]);
        __syncthreads();
        float tile = tops[par][0];
#pragma unroll
        for (int i = 1; i < kScanWaves; ++i) tile = fmaxf(tile, tops[par][i]);
        const double place = (double)tile * rate;
        if (!(place > -kReach)) {
            skipped = fmaxf(skipped, tile);
            continue;
        }
        if (place > kReach) continue;  // (the row's largest logit tells)
        const double up = (floor(__builtin_rint(place) / kOctave) + 1.0) * kOctave;
        if (!used || up > base) {
            // bins that enter at the top, where the lowest ones were
            const int by = !used || up - base >= kBins ? kBins : (int)(up - base);
            off = by == kBins ? 0 : off + by >= kBins ? off + by - kBins : off + by;
            for (int i = tid; i < by; i += kScanThreads) {
                const int b = by == kBins ? i : off - 1 - i + (off - 1 - i < 0 ? kBins : 0);
                mass[b] = 0;
                cnt[b] = 0;
            }
            base = up;
            used = true;
            __syncthreads();
        }
        const int low = (int)base - kBins;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                double past;
                int b = sample_place(fmax((double)l[k][j] * rate, base - (kBins + 1)), past) - low;
                if (b >= 0) {
                    b += off;
                    b = b >= kBins ? b - kBins : b;
                    if (by_mass) atomicAdd(&mass[b], sample_mass(past, scale));
                    atomicAdd(&cnt[b], 1u);
                }
            }
    }
    if (!cut) return;
    __syncthreads();
    SamplePart &out = p.part[(int64_t)row * p.parts + part];
    if (tid == 0) {
        out.base = base;
        out.skipped = skipped;
        out.used = used;
    }
    if (!used) return;
    for (int i = tid; i < kBins; i += kScanThreads) {
        const int b = i + off >= kBins ? i + off - kBins : i + off;
        if (by_mass) out.mass[i] = mass[b];
        out.cnt[i] = cnt[b];
    }
    if (tid < kOctaves) {
        double m = 0.0;
        uint32_t c = 0;
#pragma unroll 1
        for (int k = 0; k < kOctave; ++k) {
            const int i = tid * kOctave + k, b = i + off >= kBins ? i + off - kBins : i + off;
            if (by_mass) m += (double)mass[b] * octave[k];
            c += cnt[b];
        }
        out.octave_mass[tid] = m;
        out.octave_cnt[tid] = c;
    }
}

// ---- pick and rest: a row's token from what the scan found ----
// (62 KB: below what a launch has to ask for)
struct PickLds {
    unsigned long long mass[kBins];
    double octave[kOctave];  // the powers of 2^(1/24)
    union {
        double cmass[kChunks];
        unsigned long long rest[kChunks];  // of a list's sums
    };
    uint32_t cnt[kBins];
    float cmax[kChunks];
    float list_l[kList], sort_l[kList];
    int list_i[kList], sort_i[kList];
    int todo[kChunks];
    double scan[2][kDrawThreads / 64];
    float tops[kDrawThreads / 64], lows[kDrawThreads / 64];
    int bests[kDrawThreads / 64];
    int n_todo, n_list, n_sort, best, found_i;
    double base_cnt, base_mass;
    int ahead[kParts];  // octaves that a part's base lies below the row's; kOctaves: nothing in it
    float low[kParts];
    int bin, bin_cnt;   // of the last token that is kept
    double whole;
};

// What workgroups of a launch hand each other: past the L2 of their own, so that no fence has to
// write back and drop all of it (256 rows of 151936: 208 us a draw with fences, 90 without).
template <class T>
__device__ __forceinline__ void sample_give(T *to, T x) {
    __hip_atomic_store(to, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
__device__ __forceinline__ T sample_take(const T *from) {
    return __hip_atomic_load(from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ordered bits of a float: larger logits have larger keys
__device__ __forceinline__ uint32_t sample_key(float l) {
    const uint32_t b = __float_as_uint(l);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// the next float up or down (by 1 or -1), past -0
__device__ __forceinline__ float sample_next(float l, int by) {
    uint32_t k = sample_key(l + 0.0f) + (uint32_t)by;
    if (k == 0x7fffffffu) k += (uint32_t)by;
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// the order of the cuts: lower tokens of equal logits come first
__device__ __forceinline__ bool sample_before(float l, int i, float k, int j) { return l > k || (l == k && i < j); }
// A list's weights (up to 1, the row's largest above 1/2) as whole numbers, so that sums of a thousand
// in any order are the same: steps of 2^-53 and, of what these leave, of 2^-106, in which
// a weight of 2^-63 has 43 bits.
constexpr double kStep = 0x1p-53;
__device__ __forceinline__ unsigned long long sample_steps(double w) { return (unsigned long long)(w * 0x1p53); }
__device__ __forceinline__ unsigned long long sample_rest(double w, unsigned long long steps) {
    return (unsigned long long)((w * 0x1p53 - (double)steps) * 0x1p53);
}

// (Loops over chunks and cuts are kept rolled: the code runs once for a row, and waits
// for its own instructions too.)
// ALONE: by the differences from the largest logit, which any row's are fit for.
template <int THREADS, bool ALONE>
struct PickRow {
    static constexpr int kPickThreads = THREADS, kPickWaves = THREADS / 64;
    static constexpr int kEach = kChunks / THREADS;  // chunks of a thread
    PickLds &s;
    const SampleParams &p;
    const float *src;
    int n, chunk, chunks;
    float m;            // the largest logit
    bool flat;          // (ALONE) only logits equal to m count, all alike
    double rate, base, min_w;
    float last_l;       // the last token that is kept, in the order of the cuts
    int last_i;

    __device__ __forceinline__ PickRow(PickLds &lds, const SampleParams &params, int row)
        : s(lds), p(params), src(reinterpret_cast<const float *>(params.src + row * params.nb_src)), n(params.n_vocab), chunk(params.chunk),
          chunks(params.chunks), m(-__builtin_inff()), flat(false), rate(0.0), base(1.0), min_w(0.0), last_l(-__builtin_inff()),
          last_i(INT32_MAX) {}

    __device__ __forceinline__ double place(float l) const { return ALONE ? flat ? 0.0 : ((double)l - (double)m) * rate : (double)l * rate; }
    // the bin (below 0: none), and what is past its middle
    __device__ __forceinline__ int bin(float l, double &past) const {
        // (-inf: no place is, or at a rate of 0 none is a number)
        const int i = sample_place(fmax(place(l), base - (kBins + 1)), past) - ((int)base - kBins);
        return !ALONE || !flat || l == m ? i : -1;
    }
    __device__ __forceinline__ int bin(float l) const {
        double past;
        return bin(l, past);
    }
    __device__ __forceinline__ double weight(float l) const {
        double past;
        const int b = bin(l, past);
        return b < 0 ? 0.0 : sample_weight(s.octave, b, sample_exp(past, 1.0, 0.0));
    }
    __device__ __forceinline__ bool left_in(float l, int i) const { return !sample_before(last_l, last_i, l, i); }
    // the base of places for a largest logit within the scan's reach
    __device__ __forceinline__ void place_by_scan() { base = (floor(__builtin_rint((double)m * rate) / kOctave) + 1.0) * kOctave; }
    __device__ __forceinline__ void weights() const {
        if (threadIdx.x < kOctave) s.octave[threadIdx.x] = exp2(threadIdx.x * (1.0 / kOctave));
    }
    // the largest of a value of each wave
    __device__ __forceinline__ float over_waves(const float *v) const {
        float x = v[0];
#pragma unroll
        for (int i = 1; i < kPickWaves; ++i) x = fmaxf(x, v[i]);
        return x;
    }
    // m from the chunks' largest
    __device__ __forceinline__ void largest() {
        const int tid = threadIdx.x;
        float mine = -__builtin_inff();
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            if (tid + k * kPickThreads < chunks) mine = fmaxf(mine, s.cmax[tid + k * kPickThreads]);
        mine = wave_max(mine);
        if ((tid & 63) == 0) s.tops[tid >> 6] = mine;
        __syncthreads();
        m = over_waves(s.tops);
    }

    // Two sums over the threads in order: what is below x and y, and the whole.
    __device__ __forceinline__ void scan2(double &x, double &y, double &all_x, double &all_y) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const double ix = wave_scan(x), iy = wave_scan(y);
        __syncthreads();
        if (lane == 63) {
            s.scan[0][wave] = ix;
            s.scan[1][wave] = iy;
        }
        __syncthreads();
        double bx = 0.0, by = 0.0;
        all_x = all_y = 0.0;
#pragma unroll
        for (int i = 0; i < kPickWaves; ++i) {
            if (i == wave) {
                bx = all_x;
                by = all_y;
            }
            all_x += s.scan[0][i];
            all_y += s.scan[1][i];
        }
        x = bx + wave_before(ix);
        y = by + wave_before(iy);
    }
    __device__ __forceinline__ double scan(double x, double &all) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const double ix = wave_scan(x);
        __syncthreads();
        if (lane == 63) s.scan[0][wave] = ix;
        __syncthreads();
        double bx = 0.0;
        all = 0.0;
#pragma unroll
        for (int i = 0; i < kPickWaves; ++i) {
            if (i == wave) bx = all;
            all += s.scan[0][i];
        }
        return bx + wave_before(ix);
    }

    // The `best` (0 and above) of the last thread that has one, threads with higher ones behind
    // those with lower; -1 where none has.  (An atomic maximum of values that differ costs
    // a wave a loop over its lanes.)
    __device__ __forceinline__ int last_best(int best) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const unsigned long long b = __ballot(best >= 0);
        const int mine = b ? __builtin_amdgcn_readlane(best, 63 - __builtin_clzll(b)) : -1;
        if (lane == 0) s.bests[wave] = mine;
        __syncthreads();
        int all = s.bests[0];
#pragma unroll
        for (int i = 1; i < kPickWaves; ++i) all = s.bests[i] > all ? s.bests[i] : all;
        return all;
    }

    // The chunks that on(chunk) asks for, as a list in any order.
    template <class ON>
    __device__ __forceinline__ int ask(ON on) const {
        const int tid = threadIdx.x, lane = tid & 63;
        __syncthreads();
        if (tid == 0) s.n_todo = 0;
        __syncthreads();
#pragma unroll 1
        for (int c = tid; c - lane < chunks; c += kPickThreads) {
            const bool is = c < chunks && on(c);
            const unsigned long long b = __ballot(is);
            int at = 0;
            if (lane == 0 && b) at = atomicAdd(&s.n_todo, __builtin_popcountll(b));
            at = __builtin_amdgcn_readfirstlane(at);
            if (is) s.todo[at + __builtin_popcountll(b & ((1ull << lane) - 1))] = c;
        }
        __syncthreads();
        return s.n_todo;
    }
    // f(token, four logits from there) of the listed chunks, each chunk by one wave, the next
    // ones on their way; end(chunk) behind each chunk.
    template <class F, class END>
    __device__ __forceinline__ void each(int count, F f, END end) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int more = __builtin_ctz(chunk) - 8, subs = 1 << more;  // (chunks are 256 tokens times a power of two)
        const int mine = count > wave ? ((count - wave - 1) / kPickWaves + 1) * subs : 0;
        // two sets of registers, one on its way while the other is used
        constexpr int SET = 4;
        struct Set {
            f32x4 v[SET];
            int c[SET];
        } a, b;
        auto load = [&](Set &q, int k0) {
#pragma unroll
            for (int j = 0; j < SET; ++j) {
                const int k = k0 + j < mine ? k0 + j : mine - 1;
                q.c[j] = s.todo[wave + (k >> more) * kPickWaves];
                q.v[j] = sample_load(src, n, q.c[j] * chunk + (k & (subs - 1)) * kChunk + lane * 4);
            }
        };
        auto use = [&](const Set &q, int k0) {
#pragma unroll
            for (int j = 0; j < SET; ++j) {
                if (k0 + j >= mine) break;
                const int sub = (k0 + j) & (subs - 1);
                const int i = q.c[j] * chunk + sub * kChunk + lane * 4;
                f32x4 l = sample_fix(q.v[j], n, i);
#pragma unroll
                for (int e = 0; e < 4; ++e) l[e] = sample_clean(l[e]);
                f(i, l);
                if (sub == subs - 1) end(q.c[j]);
            }
        };
        if (mine == 0) return;
        load(a, 0);
#pragma unroll 1
        for (int k = 0; k < mine; k += 2 * SET) {
            if (k + SET < mine) load(b, k + SET);
            use(a, k);
            if (k + SET >= mine) break;
            if (k + 2 * SET < mine) load(a, k + 2 * SET);
            use(b, k + SET);
        }
    }
    // Those of a wave's four logits a lane that are in, to the list: one atomic for all.
    __device__ __forceinline__ void append(int i, f32x4 l, const bool (&in)[4]) const {
        const int lane = threadIdx.x & 63;
        unsigned long long b[4];
        int all = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            b[e] = __ballot(in[e]);
            all += __builtin_popcountll(b[e]);
        }
        if (all == 0) return;
        int at = 0;
        if (lane == 0) at = atomicAdd(&s.n_list, all);
        at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = at + __builtin_popcountll(b[e] & ((1ull << lane) - 1));
            if (in[e] && k < kList) {  // (no more are ever counted)
                s.list_l[k] = l[e];
                s.list_i[k] = i + e;
            }
            at += __builtin_popcountll(b[e]);
        }
    }
    // Of the listed chunks (of 256): the logits from `least` up and below `above` to the list,
    // the sum of w of those from `above` up to sums[chunk], where SUMS.  Four chunks of a
    // wave at a time without a branch between them, so that their chains overlap, and four
    // more on their way.
    template <bool SUMS>
    __device__ __forceinline__ void collect(int count, float least, float above, double *sums) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int mine = count > wave ? (count - wave - 1) / kPickWaves + 1 : 0;
        constexpr int SET = 4;  // (wave_sum4's)
        struct Set {
            f32x4 v[SET];
            int c[SET];
        } a, b;
        auto load = [&](Set &q, int k0) {
#pragma unroll
            for (int j = 0; j < SET; ++j) {
                const int k = k0 + j < mine ? k0 + j : mine - 1;
                q.c[j] = __builtin_amdgcn_readfirstlane(s.todo[wave + k * kPickWaves]);
                q.v[j] = sample_load(src, n, q.c[j] * kChunk + lane * 4);
            }
        };
        auto use = [&](Set &q, int k0) {
#pragma unroll
            for (int j = 0; j < SET; ++j)
                if ((q.c[j] + 1) * kChunk > n) q.v[j] = sample_fix(q.v[j], n, q.c[j] * kChunk + lane * 4);
            if (SUMS) {
                bool any = false;
#pragma unroll
                for (int j = 0; j < SET; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) any |= q.v[j][e] >= above;
                double sum[SET] = {};
                if (__any(any)) {
#pragma unroll
                    for (int j = 0; j < SET; ++j) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float l = q.v[j][e];
                            double past;
                            const int at = bin(l, past);
                            const double w = sample_weight(s.octave, at, sample_exp(past, 1.0, 0.0));
                            sum[j] += l >= above && w >= min_w ? w : 0.0;
                        }
                    }
                    sum[0] = wave_sum4(sum[0], sum[1], sum[2], sum[3]);
                }
                // (past the last one: that again)
                if ((lane & 15) == 15) sample_give(&sums[lane < 32 ? lane < 16 ? q.c[0] : q.c[2] : lane < 48 ? q.c[1] : q.c[3]], sum[0]);
            }
            unsigned long long in[SET][4];
            int all = 0;
#pragma unroll
            for (int j = 0; j < SET; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    in[j][e] = __ballot(k0 + j < mine && q.v[j][e] >= least && q.v[j][e] < above);
                    all += __builtin_popcountll(in[j][e]);
                }
            if (all == 0) return;
            int at = 0;
            if (lane == 0) at = atomicAdd(&s.n_list, all);
            at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
            for (int j = 0; j < SET; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (in[j][e] == 0) continue;
                    const int k = at + __builtin_popcountll(in[j][e] & ((1ull << lane) - 1));
                    if (((in[j][e] >> lane) & 1) && k < kList) {  // (no more are ever counted)
                        s.list_l[k] = q.v[j][e] + 0.0f;
                        s.list_i[k] = q.c[j] * kChunk + lane * 4 + e;
                    }
                    at += __builtin_popcountll(in[j][e]);
                }
        };
        if (mine == 0) return;
        load(a, 0);
#pragma unroll 1
        for (int k = 0; k < mine; k += 2 * SET) {
            if (k + SET < mine) load(b, k + SET);
            use(a, k);
            if (k + SET >= mine) break;
            if (k + 2 * SET < mine) load(a, k + 2 * SET);
            use(b, k + SET);
        }
    }

    // By one wave, from the scan's octaves and then one octave's bins: the bin of the last token
    // before which fewer than `most` tokens (by_count) or less than `most` of the whole sum of w
    // lie, its number of tokens, what lies before it, and the whole; to LDS.
    __device__ __forceinline__ void pick_scanned(const SamplePart *part, int parts, bool by_count, double most) const {
        const int lane = threadIdx.x & 63;
        const double unit = 1.0 / (double)(1ull << kMassBits);
        double base_cnt = 0.0, base_mass = 0.0, limit = most;
        int octave = 0;
#pragma unroll
        for (int level = 0; level < 2; ++level) {
            // lane: the octaves, then the octave's bins, from the highest
            const int places = level == 0 ? kOctaves : kOctave;
            double sum = 0.0, cnt = 0.0;
            uint32_t c[kParts];
            double m0[kParts];
            unsigned long long m1[kParts];
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                // (read whether or not there is any, so that all loads are on their way together)
                const int of = i < parts ? i : parts - 1, at = (level == 0 ? kOctaves - 1 - lane : octave) + s.ahead[of];
                const int o = at < kOctaves ? at : kOctaves - 1, b = o * kOctave + kOctave - 1 - (lane < kOctave ? lane : 0);
                c[i] = level == 0 ? part[of].octave_cnt[o] : part[of].cnt[b];
                if (level == 0) m0[i] = part[of].octave_mass[o];
                else m1[i] = part[of].mass[b];
            }
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                const int at = (level == 0 ? kOctaves - 1 - lane : octave) + s.ahead[i < parts ? i : 0];
                const bool is = i < parts && lane < places && at < kOctaves;
                cnt += is ? c[i] : 0;
                if (is && !by_count) sum += level == 0 ? m0[i] : (double)m1[i];
            }
            if (level == 0) sum = ldexp(sum * unit, -1 - lane);
            else if (lane < kOctave) sum = sample_weight_sum(s.octave, octave * kOctave + kOctave - 1 - lane, sum * unit);
            const double ic = wave_scan(cnt), im = wave_scan(sum);
            const double bc = base_cnt + wave_before(ic), bm = base_mass + wave_before(im);
            if (level == 0) {
                const double whole = last_lane(im);
                if (!by_count) limit = most * whole;
                if (lane == 0) s.whole = whole;
            }
            const unsigned long long b = __ballot(cnt != 0.0 && ((by_count ? bc : bm) < limit || bc == 0.0));
            const int found = 63 - __builtin_clzll(b | 1);
            base_cnt = lane_of(bc, found);
            base_mass = lane_of(bm, found);
            if (level == 0) {
                octave = kOctaves - 1 - found;
            } else if (lane == found) {
                s.bin = octave * kOctave + kOctave - 1 - found;
                s.bin_cnt = (int)cnt;
                s.base_cnt = base_cnt;
                s.base_mass = base_mass;
            }
        }
    }

    // The least logit of the bins from bin_ up, so that one comparison of F32 tells (the bins'
    // ends are steps away from their quotients by rounding only).
    __device__ __forceinline__ float least(int bin_) const {
        if (bin_ >= kBins) return __builtin_inff();
        constexpr float most = 3.4028235e38f;
        float l = (float)((base - kBins + bin_ - 0.5) / rate);
        l = l != l ? -most : fminf(fmaxf(l, -most), most);
        for (int k = 0; k < 16 && l < most && bin(l) < bin_; ++k) l = sample_next(l, 1);
        for (int k = 0; k < 16 && l > -most && bin(sample_next(l, -1)) >= bin_; ++k) l = sample_next(l, -1);
        return l;
    }

    // The bin of the last token before which fewer than `most` tokens (by_count) or
    // less than `most` of w lie, and what lies before the bin; the whole sum.  Bins from
    // the highest, a thread has as many as divide them among all; mass_of(bin): the sum of w of one that
    // is not empty.  `part`: most is of the whole.
    template <int BINS, class W>
    __device__ __forceinline__ int pick(bool by_count, bool part, double most, W mass_of, double &base_cnt, double &base_mass,
                                        double &whole) const {
        constexpr int PER = (BINS + kPickThreads - 1) / kPickThreads;
        const int tid = threadIdx.x;
        double cnt[PER], mass[PER], all, bc = 0.0, bm = 0.0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int b = BINS - 1 - (tid * PER + j);
            cnt[j] = b >= 0 ? s.cnt[b] : 0.0;
            mass[j] = cnt[j] != 0.0 ? mass_of(b) : 0.0;
            bc += cnt[j];
            bm += mass[j];
        }
        scan2(bc, bm, all, whole);
        bc += base_cnt;
        bm += base_mass;
        const double limit = part ? most * whole : most;
        int best = -1;
        double kc = 0.0, km = 0.0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            if (cnt[j] != 0.0 && ((by_count ? bc : bm) < limit || bc == 0.0)) {
                best = tid * PER + j;
                kc = bc;
                km = bm;
            }
            bc += cnt[j];
            bm += mass[j];
        }
        const int found = last_best(best);
        if (best >= 0 && found == best) {
            s.base_cnt = kc;
            s.base_mass = km;
        }
        __syncthreads();
        base_cnt = s.base_cnt;
        base_mass = s.base_mass;
        return BINS - 1 - found;
    }

    // Of tokens in order, their weights in cmass (0 behind the last), their places in cnt: the last
    // one that is kept; where `then` is 0 or above, of what was kept the last one before which less
    // than that part of it lies.  Returns the sum of w up to it.
    __device__ __forceinline__ double cut_sorted(int count, const float *list_l, const int *list_i, bool by_count, double most, double base_cnt,
                                                 double base_mass, double then) {
        const int tid = threadIdx.x;
        double w[kEach], before[kEach], mine = 0.0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            w[k] = tid * kEach + k < count ? s.cmass[tid * kEach + k] : 0.0;
            mine += w[k];
        }
        double all, at_mass = base_mass + scan(mine, all);
        const double first = base_mass + s.cmass[0];
        int found, best = tid == 0 ? 0 : -1;  // (the first one always)
        double upto = first;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int e = tid * kEach + k;
            before[k] = at_mass;
            at_mass += w[k];
            if (w[k] > 0.0 && (by_count ? base_cnt + e : before[k]) < most) {
                best = e;
                upto = at_mass;
            }
        }
        found = last_best(best);
        if (best >= 0 && best == found) s.base_mass = upto;
        if (then >= 0.0) {
            __syncthreads();
            const double limit = then * s.base_mass;
            const int last = found;
            best = tid == 0 ? 0 : -1;
            upto = first;
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                const int e = tid * kEach + k;
                if (w[k] > 0.0 && e <= last && before[k] < limit) {
                    best = e;
                    upto = before[k] + w[k];
                }
            }
            found = last_best(best);
            if (best >= 0 && best == found) s.base_mass = upto;
        }
        const int at = s.cnt[found];
        last_l = list_l[at];
        last_i = list_i[at];
        __syncthreads();
        return s.base_mass;
    }

    // Of the list's n tokens those that are left in, before which lie base_cnt and
    // base_mass: the last one that is kept becomes last_l, last_i.  Returns the sum of w
    // up to it.  `then` as above, of kShort tokens at most.
    __device__ __forceinline__ double cut_list(int n, bool by_count, double most, double base_cnt, double base_mass, double then = -1.0) {
        const int tid = threadIdx.x;
        double some;
        if (n <= kShort) {
            // every token's rank (those that are left in have keys above 0)
            if (tid < kShort) {
                const bool is = tid < n && left_in(s.list_l[tid], s.list_i[tid]);
                s.mass[tid] = is ? (unsigned long long)sample_key(s.list_l[tid]) << 32 | (uint32_t)~s.list_i[tid] : 0;
                s.cmass[tid] = 0.0;
            }
            __syncthreads();
            if (tid < n && s.mass[tid]) {
                const unsigned long long key = s.mass[tid];
                int rank = 0;
#pragma unroll 8
                for (int j = 0; j < n; ++j) rank += s.mass[j] > key;
                s.cnt[rank] = tid;
                s.cmass[rank] = weight(s.list_l[tid]);
            }
            __syncthreads();
            return cut_sorted(kShort, s.list_l, s.list_i, by_count, most, base_cnt, base_mass, then);
        }
        const int lane = tid & 63, wave = tid >> 6;
        const float inf = __builtin_inff();
        // 1024 stretches of the logits' bits between the least and the largest
        float top = -inf, low = -inf;
#pragma unroll 1
        for (int e = tid; e < n; e += kPickThreads)
            if (left_in(s.list_l[e], s.list_i[e])) {
                top = fmaxf(top, s.list_l[e]);
                low = fmaxf(low, -s.list_l[e]);
            }
        top = wave_max(top);
        low = wave_max(low);
        for (int e = tid; e < 1024; e += kPickThreads) {
            s.mass[e] = 0;
            s.cnt[e] = 0;
        }
        if (lane == 0) {
            s.tops[wave] = top;
            s.lows[wave] = low;
        }
        if (tid == 0) s.n_sort = 0;
        __syncthreads();
        const uint32_t lo = sample_key(-over_waves(s.lows)), span = (sample_key(over_waves(s.tops)) - lo) | 1023u;
        const int shift = 22 - __builtin_clz(span);
#pragma unroll 1
        for (int e = tid; e < n; e += kPickThreads) {
            const float l = s.list_l[e];
            if (!left_in(l, s.list_i[e])) continue;
            const int b = (int)((sample_key(l) - lo) >> shift);
            atomicAdd(&s.mass[b], sample_steps(weight(l)));
            atomicAdd(&s.cnt[b], 1u);
        }
        __syncthreads();
        const int sub = pick<1024>(by_count, false, most, [&](int b) { return (double)s.mass[b] * kStep; }, base_cnt, base_mass, some);
        // the tokens of that stretch in order, where the list's kept ones are looked up again
        const int count = s.cnt[sub];
#pragma unroll 1
        for (int e = tid; e < n; e += kPickThreads) {
            const float l = s.list_l[e];
            if (!left_in(l, s.list_i[e]) || (int)((sample_key(l) - lo) >> shift) != sub) continue;
            const int at = atomicAdd(&s.n_sort, 1);
            s.sort_l[at] = l;
            s.sort_i[at] = s.list_i[e];
        }
        __syncthreads();
        // (their places go to cnt, their weights in that order to cmass)
#pragma unroll 1
        for (int e = tid; e < count; e += kPickThreads) {
            const float l = s.sort_l[e];
            const int i = s.sort_i[e];
            int rank = 0;
#pragma unroll 1
            for (int j = 0; j < count; ++j) rank += sample_before(s.sort_l[j], s.sort_i[j], l, i);
            s.cnt[rank] = e;
            s.cmass[rank] = weight(l);
        }
        __syncthreads();
        return cut_sorted(count, s.sort_l, s.sort_i, by_count, most, base_cnt, base_mass, -1.0);
    }

    // The kept sums of the list's n tokens by chunks, to `have` of chunks tid * kEach ..
    __device__ __forceinline__ void list_sums(int n, double (&have)[kEach]) const {
        const int tid = threadIdx.x;
        for (int e = tid; e < kChunks; e += kPickThreads) s.mass[e] = s.rest[e] = 0;
        __syncthreads();
#pragma unroll 1
        for (int e = tid; e < n; e += kPickThreads)
            if (left_in(s.list_l[e], s.list_i[e])) {
                const double w = weight(s.list_l[e]);
                if (w >= min_w) {
                    const unsigned long long steps = sample_steps(w);
                    atomicAdd(&s.mass[s.list_i[e] / chunk], steps);
                    atomicAdd(&s.rest[s.list_i[e] / chunk], sample_rest(w, steps));
                }
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kEach; ++k) have[k] += (double)s.mass[tid * kEach + k] * kStep + (double)s.rest[tid * kEach + k] * (kStep * kStep);
    }

    // The token that u falls on, of chunks tid * kEach .. with kept sums `have`, and its share.
    __device__ __forceinline__ void draw(int row, double u, const double (&have)[kEach]) const {
        const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
        auto kept_w = [&](float l, int i) {
            const double w = weight(l);
            return left_in(l, i) && w >= min_w ? w : 0.0;
        };
        double total, mine = 0.0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) mine += have[k];
        double before = scan(mine, total);
        const double target = u * total * (1.0 + kNear);
        // the last chunk with any before which no more than the target lies
        int best = tid == 0 ? 0 : -1;
        double rest = target;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            if (have[k] > 0.0 && before <= target) {
                best = tid * kEach + k;
                rest = target - before;
            }
            before += have[k];
        }
        const int found = last_best(best);
        if (best >= 0 && best == found) s.base_mass = rest;
        __syncthreads();
        if (wave != 0) return;
        double left = s.base_mass, share = 0.0;
        const int64_t c0 = (int64_t)found * chunk;
        int token = -1;
        bool done = false;
#pragma unroll 1
        for (int64_t i = c0; i < c0 + chunk && i < n && !done; i += kChunk) {
            const int t = (int)i + lane * 4;
            const f32x4 v = sample_fix(sample_load(src, n, t), n, t);
            double w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = kept_w(sample_clean(v[j]), t + j);
            const double four = (w[0] + w[1]) + (w[2] + w[3]), inc = wave_scan(four);
            double upto = wave_before(inc), first_w = 0.0, any_w = 0.0;
            int first = -1, any = -1;  // of the lane's four, the first that passes and the last that counts
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                upto += w[j];
                if (w[j] > 0.0) {
                    any = j;
                    any_w = w[j];
                    if (upto > left && first < 0) {
                        first = j;
                        first_w = w[j];
                    }
                }
            }
            const unsigned long long passed = __ballot(first >= 0), some = __ballot(any >= 0);
            if (passed || some) {
                const int from = passed ? __builtin_ctzll(passed) : 63 - __builtin_clzll(some);
                token = (int)i + from * 4 + __shfl(passed ? first : any, from);
                share = lane_of(passed ? first_w : any_w, from);
                done = passed != 0;
            }
            left -= last_lane(inc);
        }
        if (lane == 0) {
            p.tokens[row] = token;
            if (p.logprob) p.logprob[row] = (float)log(share / total);
        }
    }

    // A row without candidates, and one whose largest logit is taken: true where that is all.
    __device__ __forceinline__ bool simple(int row, bool greedy) const {
        const int tid = threadIdx.x;
        if (m == -__builtin_inff()) {
            if (tid == 0) {
                p.tokens[row] = -1;
                if (p.logprob) p.logprob[row] = m;
            }
            return true;
        }
        if (!greedy) return false;
        const int all = ask([&](int c) { return s.cmax[c] == m; });
        int first = INT32_MAX;
        each(all, [&](int i, f32x4 l) {
#pragma unroll
            for (int e = 3; e >= 0; --e)
                if (l[e] == m && i + e < first) first = i + e;
        }, [](int) {});
        if (first != INT32_MAX) atomicMin(&s.found_i, first);
        __syncthreads();
        if (tid == 0) {
            p.tokens[row] = s.found_i;
            if (p.logprob) p.logprob[row] = 0.0f;
        }
        return true;
    }
};

// All of a row's work by one workgroup.
template <int THREADS>
__device__ __forceinline__ void sample_alone(const SampleParams &p, PickLds &s, int row) {
    using Row = PickRow<THREADS, true>;
    constexpr int kPickThreads = Row::kPickThreads, kEach = Row::kEach;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float inf = __builtin_inff();
    Row x(s, p, row);
    const SampleRules r(p, row);
    auto nothing = [](int) {};
    {
        const int all = x.ask([](int) { return true; });
        float top = -inf;
        x.each(all, [&](int, f32x4 l) { top = fmaxf(fmaxf(fmaxf(top, l[0]), fmaxf(l[1], l[2])), l[3]); },
               [&](int c) {
                   top = wave_max(top);
                   if (lane == 0) s.cmax[c] = top;
                   top = -inf;
               });
    }
    x.weights();
    if (tid == 0) s.found_i = INT32_MAX;
    __syncthreads();
    x.largest();
    if (x.simple(row, r.greedy)) return;
    x.flat = x.m == inf;  // only the infinite ones count
    x.rate = r.rate();
    const double scale = (double)(1ull << p.past_bits), unit = 1.0 / scale;
    double most = 0.0;
#pragma unroll 1
    for (int cut = r.top_k > 0 ? 0 : 1; cut < 2; ++cut) {
        if (cut == 1 && !(r.top_p < 1.0f)) break;
        const bool by_count = cut == 0, whole_row = cut == 1 && r.top_k == 0;
        const double near_p = (double)r.top_p * (1.0 - kNear);
        // the histogram of what is left in; then, as long as the bin of the last token has
        // many, that of stretches of its logits' bits (lo .. hi)
        int bin = -1;
        uint32_t lo = 0, hi = 0xffffffffu, count = 0;
        double base_cnt = 0.0, base_mass = 0.0;
        if (by_count) most = (double)r.top_k;
#pragma unroll 1
        for (;;) {
            const int shift = bin < 0 ? 0 : 22 - __builtin_clz((hi - lo) | 1023u);
            const int all = x.ask([&](int c) { return bin < 0 ? s.cmax[c] >= x.last_l : x.bin(s.cmax[c]) >= bin; });
            for (int b = tid; b < kBins; b += kPickThreads) {
                s.mass[b] = 0;
                s.cnt[b] = 0;
            }
            __syncthreads();
            x.each(all, [&](int i, f32x4 l) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    double past;
                    int b = x.bin(l[e], past);
                    if (b < 0 || !x.left_in(l[e], i + e)) continue;
                    if (bin >= 0) {
                        const uint32_t key = sample_key(l[e]);
                        if (b != bin || key < lo || key > hi) continue;
                        b = (int)((key - lo) >> shift);
                    }
                    atomicAdd(&s.mass[b], sample_past(past, scale));
                    atomicAdd(&s.cnt[b], 1u);
                }
            }, nothing);
            __syncthreads();
            // (stretches are numbered up to 1023: the bins above them are empty)
            double whole;
            const int found = x.template pick<kBins>(by_count, bin < 0 && whole_row, bin < 0 && whole_row ? near_p : most,
                                                           [&](int b) {
                                                               const double sum = (double)s.cnt[b] + (double)(long long)s.mass[b] * unit;
                                                               return sample_weight(s.octave, bin < 0 ? b : bin, sum);
                                                           }, base_cnt, base_mass, whole);
            count = s.cnt[found];
            if (bin < 0) {
                if (whole_row) most = near_p * whole;
                bin = found;
            } else {
                lo += (uint32_t)found << shift;
                if (hi - lo > (1u << shift) - 1) hi = lo + ((1u << shift) - 1);
            }
            if (count <= kList || lo == hi) break;
        }
        const int all = x.ask([&](int c) { return x.bin(s.cmax[c]) >= bin; });
        if (count <= kList) {
            if (tid == 0) s.n_list = 0;
            __syncthreads();
            x.each(all, [&](int i, f32x4 l) {
                bool in[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    in[e] = x.bin(l[e]) == bin && sample_key(l[e]) >= lo && sample_key(l[e]) <= hi && x.left_in(l[e], i + e);
                x.append(i, l, in);
            }, nothing);
            __syncthreads();
            most = near_p * x.cut_list(s.n_list, by_count, most, base_cnt, base_mass);
            continue;
        }
        // equal logits: how many of them, and the number of the last one
        const float l = __uint_as_float(lo & 0x80000000u ? lo ^ 0x80000000u : ~lo);
        const double w = x.weight(l);
        double keep = by_count ? most - base_cnt : ceil((most - base_mass) / w);
        keep = keep < 1.0 ? 1.0 : keep > count ? count : keep;
        double same = 0.0, total, mine = 0.0;
        for (int c = tid; c < kChunks; c += kPickThreads) s.cmass[c] = 0.0;
        __syncthreads();
        x.each(all, [&](int, f32x4 v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) same += v[e] == l ? 1.0 : 0.0;
        },
               [&](int c) {
                   same = wave_sum(same);
                   if (lane == 0) s.cmass[c] = same;
                   same = 0.0;
               });
        __syncthreads();
        for (int k = 0; k < kEach; ++k) mine += s.cmass[tid * kEach + k];
        double before = x.scan(mine, total);
        for (int k = 0; k < kEach; ++k) {
            const double have = s.cmass[tid * kEach + k];
            if (before < keep && before + have >= keep) {
                s.best = tid * kEach + k;
                s.base_cnt = keep - before;
            }
            before += have;
        }
        __syncthreads();
        if (wave == 0) {
            double left = s.base_cnt;
            const int64_t c0 = (int64_t)s.best * x.chunk;
#pragma unroll 1
            for (int64_t i = c0; i < c0 + x.chunk && i < x.n && left > 0.0; i += kChunk) {
                const f32x4 v = sample_fix(sample_load(x.src, x.n, (int)i + lane * 4), x.n, (int)i + lane * 4);
                double is[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) is[j] = sample_clean(v[j]) == l ? 1.0 : 0.0;
                const double four = is[0] + is[1] + is[2] + is[3], inc = wave_scan(four);
                double at = wave_before(inc);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    at += is[j];
                    if (is[j] != 0.0 && at == left) s.found_i = (int)i + lane * 4 + j;
                }
                left -= last_lane(inc);
            }
        }
        __syncthreads();
        x.last_l = l;
        x.last_i = s.found_i;
        __syncthreads();
        most = near_p * (base_mass + keep * w);
    }
    // the kept sum of each chunk
    x.min_w = (double)r.min_p * x.weight(x.m);
    const int all = x.ask([&](int c) { return s.cmax[c] >= x.last_l; });
    for (int c = tid; c < kChunks; c += kPickThreads) s.cmass[c] = 0.0;
    __syncthreads();
    double sum = 0.0, have[kEach];
    x.each(all, [&](int i, f32x4 l) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const double w = x.weight(l[e]);
            sum += w >= x.min_w && x.left_in(l[e], i + e) ? w : 0.0;
        }
    }, [&](int c) {
        sum = wave_sum(sum);
        if (lane == 0) s.cmass[c] = sum;
        sum = 0.0;
    });
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kEach; ++k) have[k] = s.cmass[tid * kEach + k];
    x.draw(row, r.u, have);
}

// What is read again of a row: nothing, the tokens from the bin up, those of the bin and the
// sums above it, the sums of all that min-p keeps; or all of it, by one workgroup.
constexpr int kNone = 0, kFew = 1, kCut = 2, kBound = 3, kAlone = 4;

__global__ __launch_bounds__(kDrawThreads) void sample_draw_kernel(SampleParams p) {
    extern __shared__ __attribute__((aligned(16))) char lds_bytes[];
    PickLds &s = *reinterpret_cast<PickLds *>(lds_bytes);
    using Row = PickRow<kDrawThreads, false>;
    constexpr int kEach = Row::kEach;
    const int tid = threadIdx.x, wave = tid >> 6;
    const int row = blockIdx.x / p.shares, share = blockIdx.x - row * p.shares;
    const float inf = __builtin_inff();
    if (p.parts == 0) {
        sample_alone<kDrawThreads>(p, s, row);
        return;
    }
    Row x(s, p, row);
    const SampleRules r(p, row);
    if (!r.cut && (r.greedy || r.min_p == 0.0f) && share != 0) return;
    const SamplePart *part = p.part + (int64_t)row * p.parts;
#pragma unroll
    for (int k = 0; k < kEach; ++k)
        if (tid + k * kDrawThreads < p.chunks) s.cmax[tid + k * kDrawThreads] = p.cmax[(int64_t)row * kChunks + tid + k * kDrawThreads];
    double part_base = 0.0;
    if (r.cut && tid < p.parts) {
        part_base = part[tid].used ? part[tid].base : -__builtin_inf();
        s.low[tid] = part[tid].skipped;
    }
    if (tid == 0) {
        s.found_i = INT32_MAX;
        s.n_list = 0;
    }
    x.weights();
    x.largest();
    if (x.m == -inf || r.greedy) {
        if (share == 0) x.simple(row, r.greedy);
        return;
    }
    x.rate = r.rate();
    // Whether the scan's places hold for this row: the largest logit within reach, nothing
    // that was left out for being too low within the bins below it.
    bool fits = fabs((double)x.m * x.rate) < kReach - kBins;
    if (fits && r.cut)
        for (int i = 0; i < p.parts; ++i)
            if (s.low[i] > -inf && ((double)x.m - (double)s.low[i]) * x.rate < 2.0 * kBins) fits = false;
    x.place_by_scan();
    x.min_w = (double)r.min_p * x.weight(x.m);
    int kind = kAlone, bin = 0;
    double most = 0.0;
    double have[kEach] = {};
    if (fits && r.cut) {
        const bool by_count = r.top_k > 0;  // (then the scan has counted only)
        const double near_p = (double)r.top_p * (1.0 - kNear);
        if (tid < p.parts) {
            const double d = (x.base - part_base) / kOctave;
            s.ahead[tid] = d < kOctaves ? (int)d : kOctaves;
        }
        // (one wave has written what it reads)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (wave == 0) x.pick_scanned(part, p.parts, by_count, by_count ? (double)r.top_k : near_p);
        __syncthreads();
        bin = s.bin;
        most = by_count ? (double)r.top_k : near_p * s.whole;
        if (s.base_cnt + s.bin_cnt <= kList) kind = kFew;
        else if (s.bin_cnt <= kList && !(by_count && r.top_p < 1.0f)) kind = kCut;
    } else if (fits && r.free()) {
        // the scan's sums of chunks, each from its own base, unless one was out of reach
        bool out = false;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const int c = tid * kEach + k;
            if (c >= p.chunks) continue;
            // (cb: one past the bin of the chunk's largest logit, which has to be numbered itself)
            const double cb = __builtin_rint((double)s.cmax[c] * x.rate) + 1.0, at = cb - x.base + kBins;
            if (!(at >= 1.0)) continue;
            out |= !(fabs(cb) < kReach);
            have[k] = sample_weight_sum(s.octave, (int)at, p.cmass[(int64_t)row * kChunks + c]);
        }
        if (out) s.n_list = 1;
        __syncthreads();
        if (s.n_list == 0) kind = kNone;
    } else if (fits) {
        // (a bin below that of the least weight that min-p keeps)
        kind = kBound;
        bin = (int)fmax(-1.0, floor(x.place(x.m) - x.base + kBins + kOctave * log2((double)r.min_p)) - 2.0);
    }
    if (kind == kAlone) {
        __syncthreads();
        if (share == 0) sample_alone<kDrawThreads>(p, s, row);
        return;
    }
    if (kind != kNone) {
        // this share's chunks of those that matter, dealt out so that each has as many
        double *cmass = p.cmass + (int64_t)row * kChunks;
        const double base_cnt = s.base_cnt, base_mass = s.base_mass;
        const float above = kind == kFew ? inf : x.least(bin + 1), least = kind == kBound ? above : x.least(bin);
        const int all = x.ask([&](int c) { return c % p.shares == share && s.cmax[c] >= least; });
        if (kind == kFew) x.template collect<false>(all, least, above, nullptr);
        else x.template collect<true>(all, least, above, cmass);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the sums are where the others will look)
        __syncthreads();
        int n = s.n_list < kList ? s.n_list : kList;  // (no more are ever counted)
        if (p.shares > 1) {
            // to the row's list; the last share to come here has them all
            SampleList &o = p.list[row];
            if (tid == 0) s.best = n ? atomicAdd(&o.n, n) : 0;
            __syncthreads();
            const int at = s.best;
            for (int e = tid; e < n && at + e < kList; e += kDrawThreads) {
                sample_give(&o.l[at + e], s.list_l[e]);
                sample_give(&o.i[at + e], s.list_i[e]);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (tid == 0) s.best = atomicAdd(&o.done, 1);
            __syncthreads();
            if (s.best != p.shares - 1) return;
            n = sample_take(&o.n);
            n = n < kList ? n : kList;
            for (int e = tid; e < n; e += kDrawThreads) {
                s.list_l[e] = sample_take(&o.l[e]);
                s.list_i[e] = sample_take(&o.i[e]);
            }
        }
        if (kind != kFew) {
#pragma unroll
            for (int k = 0; k < kEach; ++k) {
                const int c = tid * kEach + k;
                if (c < p.chunks && s.cmax[c] >= least) have[k] = sample_take(&cmass[c]);
            }
        }
        __syncthreads();
        if (kind != kBound) {
            // cut once or, where all that may be kept is in the list, twice (at once in a short one)
            const bool few = kind == kFew, both = few && r.top_k > 0 && r.top_p < 1.0f;
            const double near_p = (double)r.top_p * (1.0 - kNear);
#pragma unroll 1
            for (int cuts = both && n > kShort ? 2 : 1, k = 0; k < cuts; ++k) {
                const double kept = x.cut_list(n, r.top_k > 0 && k == 0, most, few ? 0.0 : base_cnt, few ? 0.0 : base_mass, both && n <= kShort ? near_p : -1.0);
                most = near_p * kept;
            }
            x.list_sums(n, have);
        }
    }
    x.draw(row, r.u, have);
}

// Rows of fewer than four logits, with -inf behind them, which are no candidates.
__global__ void sample_pad_kernel(SampleParams p) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (int64_t)p.n_rows * 4) return;
    const int c = (int)(i & 3);
    p.pad[i] = c < p.n_vocab ? reinterpret_cast<const float *>(p.src + (i >> 2) * p.nb_src)[c] : -__builtin_inff();
}

static_assert(sizeof(PickLds) <= 65536, "");

// How the rows are scanned: parts of them (0: not), tiles of a part.  Three workgroups a CU are there
// at once (256 rows of 151936, a call: 64 us with all cuts, with eight 67; with top-p alone 136 to 141 and 138 to 144;
// where every row has rules of its own 131 and 128).
static void sample_split(int64_t n_vocab, int64_t n_rows, int cus, int &parts, int &tiles) {
    parts = tiles = 0;
    if (n_vocab > (int64_t)kChunks * kChunk || n_vocab == 0) return;
    const int64_t all = (n_vocab + kTile - 1) / kTile;
    int64_t want = 3 * (int64_t)cus / n_rows;
    want = want < 1 ? 1 : want > kParts ? kParts : want;
    if (want > all) want = all;
    tiles = (int)((all + want - 1) / want);
    parts = (int)((all + tiles - 1) / tiles);
}
// Bytes for n_rows rows and any fewer: no split has more parts in all than this.
static size_t sample_bytes(int64_t n_vocab, int64_t n_rows, int cus) {
    if (n_vocab > (int64_t)kChunks * kChunk || n_vocab == 0) return 0;
    const int64_t most = n_rows * kParts, busy = n_rows > 3 * (int64_t)cus ? n_rows : 3 * (int64_t)cus;
    return (n_vocab < 4 ? n_rows * 16 : 0) + (size_t)((most < busy ? most : busy) * sizeof(SamplePart) + n_rows * (sizeof(SampleList) + kChunks * (sizeof(float) + sizeof(double))));
}

}  // namespace q4k

using namespace q4k;

extern "C" {

size_t q4k_sample_workspace_bytes(int64_t n_vocab, int64_t n_rows) {
    DeviceInfo *di;
    if (n_vocab < 0 || n_rows < 1 || n_vocab > (1 << 30) || !launches(n_rows, kDrawThreads) || device_info(&di) != Q4K_OK) return 0;
    return sample_bytes(n_vocab, n_rows, di->cus);
}

int q4k_sample(const float *src, int64_t n_vocab, int64_t n_rows, int64_t nb_src, const q4k_sample_rules *rules, int32_t *tokens, float *logprob,
               void *workspace, size_t workspace_bytes, void *stream) {
    if (!rules || n_vocab < 0 || n_rows < 0 || n_vocab > INT32_MAX || n_rows > INT32_MAX) return Q4K_EINVAL;
    const q4k_sample_rules &r = *rules;
    if (!aligned(src, 4) || !aligned(r.temperature, 4) || !aligned(r.top_k, 4) || !aligned(r.top_p, 4) || !aligned(r.min_p, 4) ||
        !aligned(r.uniform, 4) || !aligned(tokens, 4) || !aligned(logprob, 4))
        return Q4K_EINVAL;
    if (n_rows == 0) return Q4K_OK;
    if ((!src && n_vocab > 0) || !tokens || nb_src % 4 != 0 || (n_rows > 1 && nb_src < 4 * n_vocab)) return Q4K_EINVAL;
    if (n_vocab > (1 << 30) || !launches(n_rows, kDrawThreads)) return Q4K_EUNSUPPORTED;
    DeviceInfo *di;
    int st = device_info(&di);
    if (st != Q4K_OK) return st;
    SampleParams p{};
    p.src = reinterpret_cast<const char *>(src);
    p.nb_src = nb_src;
    p.n_vocab = (int)n_vocab;
    p.n_rows = (int)n_rows;
    p.chunk = kChunk;
    while ((n_vocab + p.chunk - 1) / p.chunk > kChunks) p.chunk *= 2;
    p.chunks = (int)((n_vocab + p.chunk - 1) / p.chunk);
    int bits = 0;
    while ((int64_t)1 << bits < n_vocab) ++bits;
    p.past_bits = 69 - bits < kMassBits ? 69 - bits : kMassBits;
    p.r = r;
    p.tokens = tokens;
    p.logprob = logprob;
    sample_split(n_vocab, n_rows, di->cus, p.parts, p.tiles);
    Workspace ws;
    st = ws.begin(workspace, workspace_bytes, sample_bytes(n_vocab, n_rows, di->cus), stream);
    if (st != Q4K_OK) return st;
    p.shares = 1;
    if (p.parts) {
        p.cmass = (double *)ws.ptr;
        p.part = (SamplePart *)(p.cmass + n_rows * kChunks);
        p.list = (SampleList *)(p.part + n_rows * p.parts);
        p.cmax = (float *)(p.list + n_rows);
        if (n_vocab < 4) {
            p.pad = p.cmax + n_rows * kChunks;
            st = launch(sample_pad_kernel, dim3((unsigned)((n_rows * 4 + 255) / 256)), 256, 0, stream, p);
            p.src = reinterpret_cast<const char *>(p.pad);
            p.nb_src = 16;
            p.n_vocab = 4;
        }
        if (st == Q4K_OK) st = launch(sample_scan_kernel, dim3((unsigned)(n_rows * p.parts)), kScanThreads, 0, stream, p);
        // Shares of 32 chunks, four a wave, or more, as many as there are at once, one a CU (256 rows of 151936:
        // one a row 131 us with top-p alone and 64 with all cuts, two 155 and 82, which were better only
        // where every row has rules of its own, 122 against 128).
        const int64_t most = (int64_t)di->cus / n_rows, want = (p.chunks + 31) / 32;
        p.shares = (int)(want < most ? want : most < 1 ? 1 : most);
        if (p.shares > kParts) p.shares = kParts;
    }
    if (st == Q4K_OK) st = launch(sample_draw_kernel, dim3((unsigned)(n_rows * p.shares)), kDrawThreads, (int)sizeof(PickLds), stream, p);
    return ws.end(st, stream);
}

}  // extern "C"

// q4k_lora.hip -- q4k_lora_add (include/q4k_batch.h): low-rank adapters, one
// per token, beside a projection that all tokens share.
//
//   h[n][j]   = sum_k x[n][k] a[i][j][k]                          (shrink), i = ids[n]
//   dst[n][m] = base[n][m] + sum_j (scale[i] h[n][j]) b[i][m][j]   (expand)
//
// Both products run on v_mfma_f32_16x16x32_bf16 over tiles of up to 64 tokens
// of one adapter: in the shrink the adapter's rows are the A operand and the
// tokens the columns of B, in the expand the rows of b and the tokens' h.  A lane
// of the result then holds four consecutive ranks (outputs) of one token.
//
// The F32 activations and h keep F32's precision: they enter as sums of three
// BF16 values (24 bits), F16 adapters as sums of two (11 bits, exact), and the
// products of all but the smallest terms are added: three matrix instructions for
// BF16 adapters, five for F16.  BF16 has F32's exponents, so nothing overflows.
//
// Memory bound: 4096 tokens of 16 adapters of rank 64, K 14336, 4096 outputs take
// 103 us (group 6, shrink 62, expand 44 one by one) where their 407 MB take 75 at a
// copy's rate.  The shrink reads its 235 MB at 3.8 TB/s; a plain read of the same
// tiles takes 40 us, the rest is its conversions and barriers at the two workgroups a
// CU that 66 KB of LDS allow (F16 adapters of ranks above 32 take 82 KB: one).  The
// expand moves its 139 MB at 3.2 TB/s: h is summed again for each chunk of outputs,
// and one step of outputs is on its way while another is computed.
// A few tokens are bound by two launches and their chains of round trips: 1 token,
// 1024 x 4096, rank 8: 5.3 + 5.5 us; 8 tokens, 14336 x 4096, rank 16: 5.5 + 6.3.
//
// A token's sums are cut by the sizes of the call and, in the direct shrink, by how
// many tokens its adapter has (to 64; of a slice of 512 where each workgroup looks
// for its tile), not by its tile: its result does not depend on which tokens share
// the tile, nor on the order in which they were put there.
#include <hip/hip_runtime.h>

#include "q4k_batch.h"
#include "q4k_device.h"

namespace q4k {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kTile = 64;        // tokens of a tile
constexpr int kSliceBallots = 8; // tokens that every workgroup looks through by itself: 8 x 64
constexpr int kSlice = 64 * kSliceBallots;

struct LoraParams {
    const char *a, *b;
    int64_t nb_a, nb_a_adapter, nb_b, nb_b_adapter;
    const float *scale;
    const int32_t *ranks;
    const char *x, *base;
    char *dst;
    int64_t nb_x, nb_base, nb_dst;
    const int32_t *ids;
    float *h;             // [ksplits][N][rp]
    const int32_t *order; // grouped: tokens by adapter, and the tiles (first, count, adapter, LoraTile::of) of them
    const int4 *tiles;
    const int32_t *n_tiles;
    int n_adapters, K, M, N, rank, rp;
    int ksplits, kchunk, mchunk;
    int enumerate;        // not grouped: blockIdx.y is a tile, not a token
    int copy;             // tokens without an adapter are copied (dst is not base)
};

struct LoraTile {
    int adapter;  // -1: tokens without one
    int count;
    int of;       // tokens of the adapter, at most a tile's: the same for its short last tile
};

// A tile's tokens into tok[0..63] (LDS), the same for all waves, and the
// workgroup's part x of `parts` of the tile's work; false: nothing to do.
// Grouped: the workgroups of an XCD (they go to the 8 XCDs in turn) take part
// after part of tiles that follow each other, so that an adapter's tiles read the
// same piece of it through one L2 (4096 tokens of 16 adapters of rank 64 and K
// 14336: 147 MB that would come from beyond it).
// Else, in the slice blockIdx.z of 512 tokens, blockIdx.y is a token, and the
// workgroup of the first, 65th, ... token of an adapter takes the 64 from there;
// or, where tiles are few against tokens, blockIdx.y is a tile that the workgroup
// counts its way to.
__device__ __forceinline__ bool lora_tile(const LoraParams &p, int parts, int *tok, LoraTile &t, int &x) {
    const int lane = threadIdx.x & 63;
    if (p.tiles) {
        const int tiles = *p.n_tiles, total = tiles * parts, id = blockIdx.x;
        if (id >= total) return false;
        const int per = total / 8, more = total % 8, xcd = id % 8;
        const int item = xcd * per + (xcd < more ? xcd : more) + id / 8;
        x = item / tiles;
        const int4 d = p.tiles[item - x * tiles];
        t.adapter = d.z;
        t.count = d.y;
        t.of = d.w;
        if (threadIdx.x < 64) tok[lane] = p.order[d.x + (lane < d.y ? lane : 0)];
        __syncthreads();
        return true;
    }
    x = blockIdx.x;
    const int base = blockIdx.z * kSlice, n = p.N - base < kSlice ? p.N - base : kSlice;
    int me = blockIdx.y;
    if (!p.enumerate && me >= n) return false;
    auto key_of = [&](int i) {
        const int id = p.ids[base + i];
        return id >= 0 && id < p.n_adapters ? id : -1;
    };
    uint64_t same[kSliceBallots];
    int before = 0, all = 0, keys[kSliceBallots];
    // (all on their way at once; past the end the last one again)
#pragma unroll
    for (int i = 0; i < kSliceBallots; ++i) keys[i] = key_of(i * 64 + lane < n ? i * 64 + lane : n - 1);
    int key;
    if (p.enumerate) {
        // blockIdx.y is the number of a tile: adapters in the order of their first tokens
        uint64_t rest[kSliceBallots];
#pragma unroll
        for (int i = 0; i < kSliceBallots; ++i) rest[i] = __ballot(i * 64 + lane < n);
        for (;;) {
            bool found = false;
            key = 0;
#pragma unroll
            for (int i = 0; i < kSliceBallots; ++i)
                if (!found && rest[i]) {
                    key = __builtin_amdgcn_readlane(keys[i], (int)__builtin_ctzll(rest[i]));
                    found = true;
                }
            if (!found) return false;
            all = 0;
#pragma unroll
            for (int i = 0; i < kSliceBallots; ++i) {
                same[i] = rest[i] & __ballot(keys[i] == key);
                all += __popcll(same[i]);
                rest[i] &= ~same[i];
            }
            const int tiles = (all + kTile - 1) / kTile;
            if (me < tiles) break;
            me -= tiles;
        }
        t.adapter = key;
        before = me * kTile;
        t.count = all - before < kTile ? all - before : kTile;
        t.of = all < kTile ? all : kTile;
        if (threadIdx.x < 64) {
            int seen = 0;
            tok[lane] = base;
#pragma unroll
            for (int i = 0; i < kSliceBallots; ++i) {
                const int pos = seen + __popcll(same[i] & ((1ull << lane) - 1)) - before;
                if ((same[i] >> lane & 1) && pos >= 0 && pos < kTile) tok[pos] = base + i * 64 + lane;
                seen += __popcll(same[i]);
            }
        }
        __syncthreads();
        return true;
    }
    key = __builtin_amdgcn_readfirstlane(key_of(me));
    t.adapter = key;
#pragma unroll
    for (int i = 0; i < kSliceBallots; ++i) {
        same[i] = __ballot(i * 64 + lane < n && keys[i] == key);
        const int d = me - i * 64;
        before += __popcll(d >= 64 ? same[i] : d > 0 ? same[i] & ((1ull << d) - 1) : 0);
        all += __popcll(same[i]);
    }
    if (before % kTile != 0) return false;
    t.count = all - before < kTile ? all - before : kTile;
    t.of = all < kTile ? all : kTile;
    if (threadIdx.x < 64) {
        tok[lane] = base + me;
        int seen = 0;
#pragma unroll
        for (int i = 0; i < kSliceBallots; ++i) {
            const int pos = seen + __popcll(same[i] & ((1ull << lane) - 1)) - before;
            if ((same[i] >> lane & 1) && pos >= 0 && pos < kTile) tok[pos] = base + i * 64 + lane;
            seen += __popcll(same[i]);
        }
    }
    __syncthreads();
    return true;
}

// Eight F32 as three BF16 vectors
__device__ __forceinline__ void bf16_terms(const float (&x)[8], bf16x8 (&t)[3]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        float r = x[j];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            t[i][j] = (__bf16)r;
            r -= (float)t[i][j];
        }
    }
}

// Eight adapter values as BF16 terms, and the sum of products with three
// activation terms: mul with the adapter as the A operand, mul_left as B
template <class T>
struct Weights;
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
template <>
struct Weights<__bf16> {
    bf16x8 w;
    __device__ __forceinline__ void set(u32x4 v) { w = __builtin_bit_cast(bf16x8, v); }
    __device__ __forceinline__ void set_terms(bf16x8 a, bf16x8) { w = a; }
    __device__ __forceinline__ bf16x8 second() const { return w; }
    __device__ __forceinline__ f32x4 mul(const bf16x8 (&x)[3], f32x4 c) const {
        return mfma(w, x[0], mfma(w, x[1], mfma(w, x[2], c)));
    }
    __device__ __forceinline__ f32x4 mul_left(const bf16x8 (&x)[3], f32x4 c) const {
        return mfma(x[0], w, mfma(x[1], w, mfma(x[2], w, c)));
    }
};
template <>
struct Weights<_Float16> {
    bf16x8 w, w2;
    __device__ __forceinline__ void set(u32x4 v) {
        const f16x8 h = __builtin_bit_cast(f16x8, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = (float)h[j];
            w[j] = (__bf16)f;
            w2[j] = (__bf16)(f - (float)w[j]);
        }
    }
    __device__ __forceinline__ void set_terms(bf16x8 a, bf16x8 b) {
        w = a;
        w2 = b;
    }
    __device__ __forceinline__ bf16x8 second() const { return w2; }
    __device__ __forceinline__ f32x4 mul(const bf16x8 (&x)[3], f32x4 c) const {
        return mfma(w, x[0], mfma(w, x[1], mfma(w2, x[0], mfma(w, x[2], mfma(w2, x[1], c)))));
    }
    __device__ __forceinline__ f32x4 mul_left(const bf16x8 (&x)[3], f32x4 c) const {
        return mfma(x[0], w, mfma(x[1], w, mfma(x[0], w2, mfma(x[2], w, mfma(x[1], w2, c)))));
    }
};

// Values [k, k + 8) of a row of n 16-bit values, zeros past its end.  VEC: n is a
// multiple of 8 and the row 16-byte aligned; else one 16-byte load of any alignment
// that ends with the row (the hardware takes them), moved into place, or single
// values in rows of fewer than eight.
template <bool VEC>
__device__ __forceinline__ u32x4 load_w(const char *row, int k, int n) {
    u32x4 v = {0, 0, 0, 0};
    if (VEC) {
        if (k < n) v = *reinterpret_cast<const u32x4 *>(row + 2 * k);
        return v;
    }
    if (n >= 8) {
        const int from = k + 8 <= n ? k : n - 8, shift = 16 * (k - from);  // shift >= 128: past the end
        __builtin_memcpy(&v, row + 2 * from, 16);
        const uint64_t w[2] = {v[0] | (uint64_t)v[1] << 32, v[2] | (uint64_t)v[3] << 32};
        const uint64_t lo = shift < 64 ? w[0] >> shift | (shift ? w[1] << (64 - shift) : 0) : shift < 128 ? w[1] >> (shift - 64) : 0;
        const uint64_t hi = shift < 64 ? w[1] >> shift : 0;
        return u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint16_t *s = reinterpret_cast<const uint16_t *>(row) + k + 2 * j;
        v[j] = (k + 2 * j < n ? s[0] : 0u) | (k + 2 * j + 1 < n ? (uint32_t)s[1] << 16 : 0u);
    }
    return v;
}
template <bool VEC>
__device__ __forceinline__ void load_x(const float *row, int k, int n, float (&x)[8]) {
    if (VEC || k + 8 <= n) {
        f32x4 v[2] = {};
        if (!VEC || k < n) {
            v[0] = *reinterpret_cast<const f32x4_any *>(row + k);
            v[1] = *reinterpret_cast<const f32x4_any *>(row + k + 4);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = v[j >> 2][j & 3];
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = k + j < n ? row[k + j] : 0.0f;
}

// the first n of eight values, zeros for the others
__device__ __forceinline__ u32x4 first_w(u32x4 v, int n) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] &= (2 * j < n ? 0xffffu : 0u) | (2 * j + 1 < n ? 0xffff0000u : 0u);
    return v;
}

// (without activations no adapter adds anything)
__device__ __forceinline__ int adapter_rank(const LoraParams &p, int i) {
    if (i < 0 || p.K == 0) return 0;
    const int r = p.ranks ? p.ranks[i] : p.rank;
    return r < 0 ? 0 : r > p.rank ? p.rank : r;
}

// How the four waves share a tile: waves over its tiles of 16 tokens, the
// others over the length (shrink: K, expand: M).  The shrink cuts its sums by it, so
// it takes the adapter's tokens for count (LoraTile::of): a short last tile has no
// more waves along K than the full ones beside it, and is done no later.
struct WaveSplit {
    int nt, part, parts;
    __device__ __forceinline__ WaveSplit(int count, int wave) {
        const int tiles = (count + 15) / 16;
        const int w = tiles <= 1 ? 1 : tiles == 2 ? 2 : 4;
        nt = wave % w;
        part = wave / w;
        parts = 4 / w;
    }
};

constexpr int kRankTiles = 4;  // rank tiles of 16 per wave: 64 ranks

// A tile's parts: K splits, groups of 16 NR ranks.
template <class T, int NR, bool VEC>
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraParams p) {
    __shared__ int tok[kTile];
    __shared__ f32x4 red[4][NR][64];
    LoraTile t;
    int part;
    if (!lora_tile(p, p.ksplits * ((p.rp + 16 * NR - 1) / (16 * NR)), tok, t, part) || t.adapter < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int ks = part % p.ksplits, j0 = part / p.ksplits * (16 * NR);
    const int r = adapter_rank(p, t.adapter);
    const WaveSplit ws(t.of, wave);
    const int token = tok[ws.nt * 16 + n];
    const float *x = reinterpret_cast<const float *>(p.x + (int64_t)token * p.nb_x);
    const char *a[NR];
    bool row[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
        const int j = j0 + i * 16 + n;
        row[i] = j < r;
        a[i] = p.a + t.adapter * p.nb_a_adapter + (row[i] ? j : 0) * p.nb_a;
    }
    f32x4 acc[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // the parts of a split take its steps of 32 in turn
    const int kend = (ks + 1) * p.kchunk < p.K ? (ks + 1) * p.kchunk : p.K;
    if (ws.nt * 16 < t.count) {
        constexpr int U = NR == 4 ? 2 : 4;  // steps in flight
        const int step = ws.parts * 32;
        for (int k0 = ks * p.kchunk + ws.part * 32; k0 < kend; k0 += step * U) {
            float xv[U][8];
            u32x4 av[U][NR];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = k0 + u * step + g * 8, n_k = k0 + u * step < kend ? p.K : 0;
                load_x<VEC>(x, k, n_k, xv[u]);
#pragma unroll
                for (int i = 0; i < NR; ++i) av[u][i] = load_w<VEC>(a[i], k, row[i] ? n_k : 0);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                bf16x8 xt[3];
                bf16_terms(xv[u], xt);
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    Weights<T> w;
                    w.set(av[u][i]);
                    acc[i] = w.mul(xt, acc[i]);
                }
            }
        }
    }
    if (ws.parts > 1) {
#pragma unroll
        for (int i = 0; i < NR; ++i) red[wave][i][lane] = acc[i];
        __syncthreads();
        if (ws.part != 0) return;
        for (int w = 1; w < ws.parts; ++w)
#pragma unroll
            for (int i = 0; i < NR; ++i) acc[i] += red[wave + w * (4 / ws.parts)][i][lane];
    }
    if (ws.nt * 16 + n >= t.count) return;
    float *h = p.h + ((int64_t)ks * p.N + token) * p.rp + j0 + g * 4;
#pragma unroll
    for (int i = 0; i < NR; ++i)
        if (j0 + i * 16 < p.rp) *reinterpret_cast<f32x4 *>(h + i * 16) = acc[i];
}

// The same for tiles of many tokens: activations and adapter rows come from
// memory side by side, 64 values of K at a time, and pass through LDS -- the
// activations as their three BF16 terms, F16 adapter rows as their two -- so each
// value is converted once and the waves, one per 16 tokens, share the adapter.
template <class T>
struct LdsTerms {
    static constexpr int n = __is_same(T, _Float16) ? 2 : 1;  // BF16 values of an adapter's value
};
template <class T, int NR>
__global__ __launch_bounds__(256) void lora_shrink_tiled_kernel(LoraParams p) {
    constexpr int KT = 64, CH = KT / 8, WT = LdsTerms<T>::n, NA = NR * 16 * CH;  // NA: 16-byte pieces of the adapter's tile
    __shared__ int tok[kTile];
    // two tiles: one is multiplied while the next one is written
    __shared__ __attribute__((aligned(16))) __bf16 xs2[2][3][kTile * KT], as2[2][WT][NR * 16 * KT];
    LoraTile t;
    int part;
    if (!lora_tile(p, p.ksplits * ((p.rp + 16 * NR - 1) / (16 * NR)), tok, t, part) || t.adapter < 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int ks = part % p.ksplits, j0 = part / p.ksplits * (16 * NR);
    const int r = adapter_rank(p, t.adapter);
    const int kend = (ks + 1) * p.kchunk < p.K ? (ks + 1) * p.kchunk : p.K;
    // chunk c of row t at c ^ (t / 2 % 8): 16 lanes that read the same chunk of 16 rows meet no bank twice
    auto at = [](int row, int c) { return (row * CH + (c ^ ((row >> 1) & 7))) * 8; };
    // thread: activations xk.. of the tile's rows tid / 16 + 16 i, 8 values ac of adapter rows tid / 8 + 32 i
    constexpr int XI = 4, AI = (NA + 255) / 256;
    const int xk = tid % 16 * 4, ac = tid % CH;
    const float *xp[XI];
    const char *ap[AI];
    bool arow[AI];
#pragma unroll
    for (int i = 0; i < XI; ++i) {
        const int row = tid / 16 + 16 * i;
        xp[i] = reinterpret_cast<const float *>(p.x + (int64_t)tok[row < t.count ? row : 0] * p.nb_x);
    }
#pragma unroll
    for (int i = 0; i < AI; ++i) {
        const int j = j0 + tid / CH + 32 * i;
        arow[i] = j < r && tid / CH + 32 * i < 16 * NR;
        ap[i] = p.a + t.adapter * p.nb_a_adapter + (arow[i] ? j : 0) * p.nb_a;
    }
    f32x4 xb[2][XI];  // two tiles on their way
    u32x4 ab[2][AI];
    // (No branches, or the waits for these loads would be for all of them: past the
    // end the split's first values again, taken for zeros when they are used.)
    const int k_first = ks * p.kchunk;
    auto load = [&](int k0, f32x4 (&xv)[XI], u32x4 (&av)[AI]) {
        const int xo = k0 + xk < kend ? k0 + xk : k_first, ao = 2 * (k0 + ac * 8 < kend ? k0 + ac * 8 : k_first);
#pragma unroll
        for (int i = 0; i < XI; ++i) xv[i] = load4<true>(xp[i] + xo);
#pragma unroll
        for (int i = 0; i < AI; ++i) av[i] = *reinterpret_cast<const u32x4 *>(ap[i] + ao);
    };
    f32x4 acc[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    auto write = [&](int k0, const f32x4 (&xv)[XI], const u32x4 (&av)[AI], __bf16 (&xs)[3][kTile * KT], __bf16 (&as)[WT][NR * 16 * KT]) {
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
            bf16x4 tm[3];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float y = k0 + xk < kend ? xv[i][j] : 0.0f;
#pragma unroll
                for (int e = 0; e < 3; ++e) {
                    tm[e][j] = (__bf16)y;
                    y -= (float)tm[e][j];
                }
            }
            const int o = at(tid / 16 + 16 * i, xk / 8) + (xk & 4);
#pragma unroll
            for (int e = 0; e < 3; ++e) *reinterpret_cast<bf16x4 *>(xs[e] + o) = tm[e];
        }
#pragma unroll
        for (int i = 0; i < AI; ++i) {
            const int row = tid / CH + 32 * i;
            if (NA % 256 != 0 && row >= 16 * NR) continue;
            Weights<T> w;
            w.set(k0 + ac * 8 < kend && arow[i] ? av[i] : u32x4{0, 0, 0, 0});
            *reinterpret_cast<bf16x8 *>(as[0] + at(row, ac)) = w.w;
            if (WT > 1) *reinterpret_cast<bf16x8 *>(as[WT - 1] + at(row, ac)) = w.second();
        }
    };
    auto multiply = [&](const __bf16 (&xs)[3][kTile * KT], const __bf16 (&as)[WT][NR * 16 * KT]) {
        if (wave * 16 < t.count) {
#pragma unroll
            for (int kk = 0; kk < KT / 32; ++kk) {
                bf16x8 xt[3];
#pragma unroll
                for (int e = 0; e < 3; ++e) xt[e] = *reinterpret_cast<const bf16x8 *>(xs[e] + at(wave * 16 + n, kk * 4 + g));
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    Weights<T> w;
                    w.set_terms(*reinterpret_cast<const bf16x8 *>(as[0] + at(i * 16 + n, kk * 4 + g)),
                                *reinterpret_cast<const bf16x8 *>(as[WT - 1] + at(i * 16 + n, kk * 4 + g)));
                    acc[i] = w.mul(xt, acc[i]);
                }
            }
        }
    };
    load(k_first, xb[0], ab[0]);
    load(k_first + KT, xb[1], ab[1]);
    write(k_first, xb[0], ab[0], xs2[0], as2[0]);
    load(k_first + 2 * KT, xb[0], ab[0]);
    __syncthreads();
    for (int k0 = k_first; k0 < kend; k0 += 2 * KT) {
        // tile k0 is in LDS 0; k0 + KT in registers 1, k0 + 2 KT in registers 0
        write(k0 + KT, xb[1], ab[1], xs2[1], as2[1]);
        load(k0 + 3 * KT, xb[1], ab[1]);
        multiply(xs2[0], as2[0]);
        __syncthreads();
        write(k0 + 2 * KT, xb[0], ab[0], xs2[0], as2[0]);
        load(k0 + 4 * KT, xb[0], ab[0]);
        multiply(xs2[1], as2[1]);
        __syncthreads();
    }
    if (wave * 16 + n >= t.count) return;
    float *h = p.h + ((int64_t)ks * p.N + tok[wave * 16 + n]) * p.rp + j0 + g * 4;
#pragma unroll
    for (int i = 0; i < NR; ++i)
        if (j0 + i * 16 < p.rp) *reinterpret_cast<f32x4 *>(h + i * 16) = acc[i];
}

// KR: steps of 32 ranks; VB: rows of b in aligned 16-byte loads.  The tokens are
// the A operand here: a lane of a result has one output of four tokens.  Of the
// four tiles that are in flight, lane n's outputs are 4 n .. 4 n + 3, so that 16
// lanes store 256 bytes of a token side by side.
// NT: base and dst past the caches, where they are larger than the L2s.
template <class T, int KR, bool VB, bool NT>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraParams p) {
    __shared__ int tok[kTile];
    LoraTile t;
    int part;
    if (!lora_tile(p, (p.M + p.mchunk - 1) / p.mchunk, tok, t, part) || (t.adapter < 0 && !p.copy)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int r = adapter_rank(p, t.adapter);
    const WaveSplit ws(t.count, wave);  // (waves without tokens take the first one along and store nothing)
    constexpr bool SH = KR <= 2;  // h's terms in LDS (24 KB at 64 ranks)
    __shared__ bf16x8 hs[3][SH ? kTile * KR * 4 : 1];
    const float *base[4];
    float *dst[4];
    bool live[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        live[j] = ws.nt * 16 + g * 4 + j < t.count;
        const int64_t token = tok[live[j] ? ws.nt * 16 + g * 4 + j : 0];
        base[j] = reinterpret_cast<const float *>(p.base + token * p.nb_base);
        dst[j] = reinterpret_cast<float *>(p.dst + token * p.nb_dst);
    }
    const char *b = p.b + (t.adapter < 0 ? 0 : t.adapter) * p.nb_b_adapter;
    const int m0 = part * p.mchunk, m1 = m0 + p.mchunk < p.M ? m0 + p.mchunk : p.M;
    constexpr int U = 4;  // tiles of 16 outputs in flight
    const int step = ws.parts * 16 * U;
    u32x4 bv[U][KR];
    f32x4 y[4];
    auto load = [&](int mb) {
        // (rows of b clamped; only whole fours of a row in one access)
        const int m = mb + n * U;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int kk = 0; kk < KR; ++kk) bv[u][kk] = load_w<VB>(b + (m + u < m1 ? m + u : m0) * p.nb_b, kk * 32 + g * 8, r);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (!p.base) return;
        if (m + U <= m1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = load4<NT>(base[j] + m);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (m + u < m1) y[j][u] = base[j][m + u];
        }
    };
    int mb = m0 + ws.part * 16 * U;
    if (mb < m1) load(mb);
    // h, while the first outputs' values are on their way
    bf16x8 ht[KR][3];
    const float scale = p.scale && r > 0 ? p.scale[t.adapter] : 1.0f;  // (of rank 0 it may be alpha / 0)
    if (SH) {
        // whole rows of h side by side, summed over the splits and turned into terms once per workgroup
        constexpr int CH = KR * 4;  // pieces of eight ranks
        const int tiles = (t.count + 15) / 16;
        for (int x = threadIdx.x; x < tiles * 16 * CH; x += 256) {
            const int row = x / CH, c = x % CH;
            float hv[8] = {};
            if (row < t.count && c * 8 < r) {  // (rp is a multiple of 16, so eight ranks are there or not)
#pragma unroll 4
                for (int s = 0; s < p.ksplits; ++s) {
                    const f32x4 *h = reinterpret_cast<const f32x4 *>(p.h + ((int64_t)s * p.N + tok[row]) * p.rp + c * 8);
                    const f32x4 h0 = h[0], h1 = h[1];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        hv[e] += h0[e];
                        hv[e + 4] += h1[e];
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) hv[e] *= scale;
            bf16x8 tm[3];
            bf16_terms(hv, tm);
#pragma unroll
            for (int e = 0; e < 3; ++e) hs[e][row * CH + (c ^ (row & (CH - 1)))] = tm[e];
        }
        __syncthreads();
        if (ws.nt * 16 >= t.count) return;
#pragma unroll
        for (int kk = 0; kk < KR; ++kk)
#pragma unroll
            for (int e = 0; e < 3; ++e) ht[kk][e] = hs[e][(ws.nt * 16 + n) * CH + ((kk * 4 + g) ^ (n & (CH - 1)))];
    } else {
        if (ws.nt * 16 >= t.count) return;
        const int mine = tok[ws.nt * 16 + n];
#pragma unroll
        for (int kk = 0; kk < KR; ++kk) {
            float hv[8] = {};
            const int j = kk * 32 + g * 8;
            if (j < r)
                for (int s = 0; s < p.ksplits; ++s) {
                    const float *h = p.h + ((int64_t)s * p.N + mine) * p.rp + j;
                    const f32x4 h0 = *reinterpret_cast<const f32x4 *>(h), h1 = *reinterpret_cast<const f32x4 *>(h + 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        hv[e] += h0[e];
                        hv[e + 4] += h1[e];
                    }
                }
#pragma unroll
            for (int e = 0; e < 8; ++e) hv[e] *= scale;
            bf16_terms(hv, ht[kk]);
        }
    }
    for (; mb < m1; mb += step) {
        f32x4 out[4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kk = 0; kk < KR; ++kk) {
                Weights<T> w;
                if (VB && (r & 7)) bv[u][kk] = first_w(bv[u][kk], r - kk * 32 - g * 8);
                w.set(bv[u][kk]);
                acc = w.mul_left(ht[kk], acc);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j][u] = y[j][u] + acc[j];
        }
        if (mb + step < m1) load(mb + step);
        const int m = mb + n * U;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (!live[j]) continue;
            if (m + U <= m1) {
                store4<NT>(dst[j] + m, out[j]);
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (m + u < m1) dst[j][m + u] = out[j][u];
            }
        }
    }
}

// Tokens by adapter (counting sort in LDS, one workgroup) and the tiles of up to
// 64 of them.  Atomics order the tokens within an adapter, on which no result
// depends.
__global__ __launch_bounds__(1024) void lora_group_kernel(LoraParams p) {
    extern __shared__ int lds[];
    const int keys = p.n_adapters + 1, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int *start = lds;                  // counts, then where each adapter's tokens go next
    int *wsum = lds + keys;            // [2][16]
    int32_t *order = const_cast<int32_t *>(p.order);
    int4 *tiles = const_cast<int4 *>(p.tiles);
    auto key_of = [&](int i) {
        const int id = i < p.N ? p.ids[i] : -1;
        return id >= 0 && id < p.n_adapters ? id : p.n_adapters;
    };
    int key[4];  // the first 4096 tokens' keys stay in registers
#pragma unroll
    for (int u = 0; u < 4; ++u) key[u] = key_of(u * 1024 + tid);
    // The lane's place after what was counted before.  In prompts the 64 lanes hold
    // one key, which the first lane counts for all that hold its own; the others count
    // themselves (an atomic per key in turn: 2414 tokens of 37 adapters 27 us).
    auto count = [&](int k, bool in) {
        const uint64_t any = __ballot(in);
        const int first = any ? (int)__builtin_ctzll(any) : 0;
        const int k0 = __builtin_amdgcn_readlane(k, first);
        const bool with = in && k == k0;
        const uint64_t same = __ballot(with);
        int old = 0;
        if (with ? lane == first : in) old = atomicAdd(&start[k], with ? (int)__popcll(same) : 1);
        const int old0 = __builtin_amdgcn_readlane(old, first);
        return with ? old0 + (int)__popcll(same & ((1ull << lane) - 1)) : old;
    };
    const int upto = (p.N + 1023) / 1024 * 1024;
    for (int i = tid; i < keys; i += 1024) start[i] = 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) count(key[u], u * 1024 + tid < p.N);
    for (int i = 4096 + tid; i < upto; i += 1024) count(key_of(i), i < p.N);
    __syncthreads();
    // scan of the counts and of the numbers of tiles, 1024 keys at a time
    int tokens = 0, ntiles = 0;
    for (int k0 = 0; k0 < keys; k0 += 1024) {
        const int k = k0 + tid;
        const int c = k < keys ? start[k] : 0, q = (c + kTile - 1) / kTile;
        int sc = c, sq = q;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int a = __shfl_up(sc, d), b = __shfl_up(sq, d);
            if (lane >= d) {
                sc += a;
                sq += b;
            }
        }
        if (lane == 63) {
            wsum[wave] = sc;
            wsum[16 + wave] = sq;
        }
        __syncthreads();
        int bc = tokens, bq = ntiles, tc = 0, tq = 0;
        for (int w = 0; w < 16; ++w) {
            if (w < wave) {
                bc += wsum[w];
                bq += wsum[16 + w];
            }
            tc += wsum[w];
            tq += wsum[16 + w];
        }
        const int first = bc + sc - c;
        for (int i = 0; i < q; ++i)
            tiles[bq + sq - q + i] = make_int4(first + i * kTile, c - i * kTile < kTile ? c - i * kTile : kTile,
                                               k < p.n_adapters ? k : -1, c < kTile ? c : kTile);
        if (k < keys) start[k] = first;
        tokens += tc;
        ntiles += tq;
        __syncthreads();
    }
    if (tid == 0) *const_cast<int32_t *>(p.n_tiles) = ntiles;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int i = u * 1024 + tid, at = count(key[u], i < p.N);
        if (i < p.N) order[at] = i;
    }
    for (int i = 4096 + tid; i < upto; i += 1024) {
        const int at = count(key_of(i), i < p.N);
        if (i < p.N) order[at] = i;
    }
}

// ---------------------------------------------------------------- host ----

struct LoraPlan {
    bool grouped, tiled;
    int rows;           // not grouped: workgroups in y, one per tile if enumerate
    bool enumerate;
    int max_tiles;      // tiles there can be, grouped
    int rp, nr, ksplits, kchunk, mchunk;
    size_t h_bytes, bytes;
    size_t upto_bytes;  // enough for this many tokens and for any fewer
};

constexpr int kGroupKeys = 32000;  // counters in the group kernel's LDS

static int lora_plan(const q4k_lora &l, int64_t K, int64_t M, int64_t N, LoraPlan &pl) {
    constexpr int64_t cus = 256;
    if (K > 1 << 30) return Q4K_EUNSUPPORTED;  // the kernels count a 16-bit row's bytes in 31 bits
    pl.grouped = N > kSlice && l.n_adapters < kGroupKeys;
    const int64_t kinds = l.n_adapters + 1 < N ? l.n_adapters + 1 : N;
    const int64_t tiles = N / kTile + kinds;  // at most
    pl.max_tiles = (int)tiles;
    pl.tiled = N >= 16 * kinds;
    // Counting to a tile takes about 0.1 us for each adapter before it, a workgroup
    // for a token that leads no tile 1.5 us of its place: counted where there are
    // sixteen tokens and more a tile.
    const int64_t in_slice = N < kSlice ? N : kSlice, slice_tiles = in_slice / kTile + (kinds < in_slice ? kinds : in_slice);
    pl.enumerate = slice_tiles * 16 <= in_slice;
    pl.rows = (int)(pl.enumerate ? slice_tiles : in_slice);
    pl.rp = (l.rank + 15) / 16 * 16;
    pl.nr = pl.rp / 16 < kRankTiles ? pl.rp / 16 : kRankTiles;
    if (pl.nr == 3) pl.nr = 4;
    const int64_t groups = (pl.rp + 16 * pl.nr - 1) / (16 * pl.nr);
    // Two workgroups per CU, in splits that every workgroup of the expand reads again:
    // of tiled loads at most 32 and at least 256 values (us at most 8 of 512 / 16 / 32:
    // one tile of 64 tokens, K 14336, rank 16: 29.4 / 20.6 / 17.4; 8 tiles 32.6 / 23.9 /
    // 22.5), of direct ones, whose workgroups share less work, 8 and 512 values (48
    // tokens of 32 adapters, K 8192: 13.9 / 15.6 / 15.7).
    int64_t ks = 2 * cus / (tiles * groups);
    const int64_t most = pl.tiled ? (K / 256 < 32 ? K / 256 : 32) : K / 512 < 8 ? K / 512 : 8;
    ks = ks > most ? most : ks;
    ks = ks < 1 ? 1 : ks;
    pl.kchunk = (int)(((K + ks - 1) / ks + 127) / 128 * 128);
    if (pl.kchunk < 128) pl.kchunk = 128;
    pl.ksplits = K > 0 ? (int)((K + pl.kchunk - 1) / pl.kchunk) : 0;
    // Two workgroups per CU, at least one row tile per wave.  At most 1024 outputs, as
    // each reads its tokens' h first (4096 tokens of 16 adapters of rank 64: 103 us, of
    // 512 outputs 107), and 512 where that is little (2414 tokens of 37 adapters of rank
    // 16 x 12032 outputs: 86.5 / 78.2 us).
    const int64_t widest = pl.tiled && l.rank <= 32 ? 512 : 1024;
    int64_t mc = (M * tiles / (2 * cus) + 63) / 64 * 64;
    mc = mc < 64 ? 64 : mc > widest ? widest : mc;
    pl.mchunk = (int)mc;
    if (N > ((int64_t)1 << 50) / (pl.rp * 4 * 32)) return Q4K_EUNSUPPORTED;
    pl.h_bytes = (size_t)((int64_t)pl.ksplits * N * pl.rp * 4 + 15) / 16 * 16;
    const size_t group_bytes = pl.grouped ? (size_t)tiles * 16 + (size_t)N * 4 + 16 : 0;
    pl.bytes = pl.h_bytes + group_bytes;
    // Fewer tokens take more splits of K each.  n tokens are more than n / 64 tiles, so
    // ks n <= 2 cus n / (tiles groups) < 128 cus / groups where there is more than one
    // split, and there are no more splits than `most` may be.
    const int64_t max_splits = K / 256 < 1 ? 1 : K / 256 < 32 ? K / 256 : 32;
    int64_t split_rows = max_splits * N < 128 * cus / groups ? max_splits * N : 128 * cus / groups;
    split_rows = K == 0 ? 0 : split_rows < N ? N : split_rows;
    pl.upto_bytes = (size_t)(split_rows * pl.rp * 4) + group_bytes;
    return Q4K_OK;
}

static bool lora_sizes_ok(const q4k_lora *l, int64_t ne00, int64_t ne01, int64_t ne11) {
    return l && (l->type == Q4K_GGML_TYPE_F16 || l->type == Q4K_GGML_TYPE_BF16) && l->rank >= 1 &&
           l->rank <= Q4K_LORA_MAX_RANK && l->n_adapters >= 0 && l->n_adapters <= INT32_MAX - 2 && ne00 >= 0 && ne01 >= 0 &&
           ne11 >= 0 && ne00 <= INT32_MAX - 4096 && ne01 <= INT32_MAX - 4096 && ne11 <= INT32_MAX - 4096;
}

using LoraFn = void (*)(LoraParams);

template <class T, bool VEC>
LoraFn shrink_of(int nr) {
    return nr == 1 ? lora_shrink_kernel<T, 1, VEC> : nr == 2 ? lora_shrink_kernel<T, 2, VEC> : lora_shrink_kernel<T, 4, VEC>;
}
template <class T>
LoraFn tiled_of(int nr) {
    return nr == 1 ? lora_shrink_tiled_kernel<T, 1> : nr == 2 ? lora_shrink_tiled_kernel<T, 2> : lora_shrink_tiled_kernel<T, 4>;
}
template <class T, bool VB, bool NT>
LoraFn expand_of(int kr) {
    return kr <= 1   ? lora_expand_kernel<T, 1, VB, NT>
           : kr <= 2 ? lora_expand_kernel<T, 2, VB, NT>
           : kr <= 4 ? lora_expand_kernel<T, 4, VB, NT>
                     : lora_expand_kernel<T, 8, VB, NT>;
}
template <class T>
LoraFn expand_of(int kr, bool vb, bool nt) {
    return vb ? (nt ? expand_of<T, true, true>(kr) : expand_of<T, true, false>(kr))
              : (nt ? expand_of<T, false, true>(kr) : expand_of<T, false, false>(kr));
}

}  // namespace q4k

using namespace q4k;

extern "C" {

size_t q4k_lora_workspace_bytes(const q4k_lora *lora, int64_t ne00, int64_t ne01, int64_t ne11) {
    LoraPlan pl;
    if (!lora_sizes_ok(lora, ne00, ne01, ne11) || ne11 == 0 || lora_plan(*lora, ne00, ne01, ne11, pl) != Q4K_OK) return 0;
    return pl.upto_bytes;
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
        if ((ne00 > 0 && !l.a) || !l.b) return Q4K_EINVAL;
        if (l.nb_a % 2 != 0 || l.nb_b % 2 != 0 || l.nb_a_adapter % 2 != 0 || l.nb_b_adapter % 2 != 0) return Q4K_EINVAL;
        if (l.nb_a < 2 * ne00 || l.nb_b < 2 * l.rank || l.nb_a_adapter < 0 || l.nb_b_adapter < 0) return Q4K_EINVAL;
    }
    LoraPlan pl;
    int st = lora_plan(l, ne00, ne01, ne11, pl);
    if (st != Q4K_OK) return st;
    DeviceInfo *di;
    st = device_info(&di);
    if (st != Q4K_OK) return st;
    const int64_t slices = (ne11 + kSlice - 1) / kSlice;
    const int64_t parts1 = (int64_t)pl.ksplits * ((pl.rp + 16 * pl.nr - 1) / (16 * pl.nr)), parts2 = (ne01 + pl.mchunk - 1) / pl.mchunk;
    const int64_t most = parts1 > parts2 ? parts1 : parts2;
    if (pl.grouped ? pl.max_tiles > INT32_MAX / most : slices > 65535) return Q4K_EUNSUPPORTED;
    Workspace ws;
    st = ws.begin(workspace, workspace_bytes, pl.bytes, stream);
    if (st != Q4K_OK) return st;
    LoraParams p{};
    p.a = (const char *)l.a; p.b = (const char *)l.b;
    p.nb_a = l.nb_a; p.nb_a_adapter = l.nb_a_adapter; p.nb_b = l.nb_b; p.nb_b_adapter = l.nb_b_adapter;
    p.n_adapters = (int)l.n_adapters; p.scale = l.scale; p.ranks = l.ranks;
    p.x = (const char *)src1; p.base = (const char *)src2; p.dst = (char *)dst;
    p.nb_x = nb11; p.nb_base = nb21; p.nb_dst = nb1;
    p.ids = ids; p.h = (float *)ws.ptr; p.K = (int)ne00; p.M = (int)ne01; p.N = (int)ne11;
    p.rank = l.rank; p.rp = pl.rp; p.ksplits = pl.ksplits; p.kchunk = pl.kchunk; p.mchunk = pl.mchunk;
    p.copy = src2 != dst;
    p.enumerate = pl.enumerate;
    dim3 grid;
    auto grid_of = [&](int64_t parts) {
        return pl.grouped ? dim3((unsigned)(parts * pl.max_tiles))
                          : dim3((unsigned)parts, (unsigned)pl.rows, (unsigned)slices);
    };
    if (pl.grouped) {
        char *w = (char *)ws.ptr + pl.h_bytes;
        p.tiles = (const int4 *)w;
        p.order = (const int32_t *)(w + (size_t)pl.max_tiles * 16);
        p.n_tiles = p.order + ne11;
        const int lds = (int)(l.n_adapters + 1 + 32) * 4;
        st = ensure_lds(di, (const void *)&lora_group_kernel, lds);
        if (st == Q4K_OK) st = launch(lora_group_kernel, dim3(1), 1024, lds, stream, p);
    }
    const bool f16 = l.type == Q4K_GGML_TYPE_F16;
    if (st == Q4K_OK && pl.ksplits > 0 && l.n_adapters > 0) {
        const bool vec = ne00 % 8 == 0 && aligned(l.a, 16) && (l.nb_a | l.nb_a_adapter) % 16 == 0 && aligned(src1, 16) &&
                         nb11 % 16 == 0;
        grid = grid_of(parts1);
        // many tokens of an adapter to a tile: through LDS, else straight to the operands
        const LoraFn fn = vec && pl.tiled ? (f16 ? tiled_of<_Float16>(pl.nr) : tiled_of<__bf16>(pl.nr))
                          : vec           ? (f16 ? shrink_of<_Float16, true>(pl.nr) : shrink_of<__bf16, true>(pl.nr))
                                          : (f16 ? shrink_of<_Float16, false>(pl.nr) : shrink_of<__bf16, false>(pl.nr));
        st = launch(fn, grid, 256, 0, stream, p);
    }
    if (st == Q4K_OK) {
        const bool vb = l.rank % 8 == 0 && aligned(l.b, 16) && (l.nb_b | l.nb_b_adapter) % 16 == 0;
        grid = grid_of(parts2);
        const int kr = (l.rank + 31) / 32;
        // (rows that begin inside a cache line would write their ends past the caches in
        // parts: 4089 tokens of 13249 outputs 219 us against 187)
        const bool nt = ne11 * ne01 >= kStreamFloats && aligned(dst, 64) && nb1 % 64 == 0;
        st = launch(f16 ? expand_of<_Float16>(kr, vb, nt) : expand_of<__bf16>(kr, vb, nt), grid, 256, 0, stream, p);
    }
    return ws.end(st, stream);
}

}  // extern "C"

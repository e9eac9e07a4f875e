// q4k_kv8_attn.h -- the attention kernel over paged caches of 8 bits
// (q4k_kv8_attn.hip).
//
// A workgroup takes up to 16 * RT query rows (token, head of the group) of one
// request and KV head and a stretch of its positions; its four waves go over steps
// of 32 positions of their own, once, with a running maximum and sum, and join at
// the end:
//   S^T = (K Q^T) ks      v_mfma_f32_16x16x32 on the bytes as F16 (BF16), exact
//   P = exp2(c S - M)     in the lanes that hold S
//   O^T += V^T (P vs)^T   v_mfma_f32_16x16x32_bf16, P vs as 2 or 3 BF16 terms
// Nothing passes through LDS on the way.  The sums over dimensions (K Q^T) and
// positions (V^T P^T) may take theirs in any order that both operands share, so
// each lane reads what it has to hold, in whole rows of a head:
//   K  lane (n, g): 16 bytes of a row at g * 16, which are its operands of two
//      products; row n of tile tt is position (n / 4) * 8 + tt * 4 + n % 4 of the step
//   P  so that a lane's eight scores are those of positions g * 8 .. g * 8 + 7
//   V  lane (n, g): D / 16 bytes at n * D / 16 of these eight positions, byte dt of
//      which belongs to tile dt of the output
// A lane's eight positions share a page and, where blocks are multiples of eight
// tokens, a scale.
//
// Long caches are bound by memory: 64 requests of 512 to 8192 positions, 8 heads of 128 e4m3, 680 MB,
// BF16 queries of 64 heads, 147 us, 4.6 TB/s, what large reads reach here.  16 of them with F32 queries,
// 175 MB of int8, 48 us and 6 us of join, of which 8 us pass before the first step (lengths counted, page,
// first positions); two steps on their way a wave: 51 us.  One request of 200: 9 us, a chain.
// Prompts are bound by arithmetic, of which a tile of 32 rows does all that its request has, also what lies behind its
// causal bound, and every tile converts every byte again: the first 2048 tokens of 32/8 heads of 128, BF16 on e4m3,
// 218 us, 158 TFLOP/s of what the rows see, the second 2048 339 us, 304.
#pragma once

#include "q4k_attn.h"
#include "q4k_join.h"
#include "q4k_kv8.h"
#include "q4k_scan.h"

namespace q4k {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct Kv8AttnParams {
    AttnParams a;  // rows and partial results; `suf` parts only, no AttnCache
    Kv8Cache c;
    // (a.join stays 0: attn_emit writes dst.)
    int each;       // steps of a part of a tile's positions, where parts are of one length
    int shares;     // workgroups that all steps are dealt out to (else 0), and the number of steps
    double *starts; // before each request's and, last, of all, for the join
};

// Positions of a step of four waves; the least steps of a part (200 positions of one request: 1 step a
// part and a join 14.0 us, 2 11.4), the most of parts of one length.  Parts against steps dealt out, us, BF16 on
// e4m3: 2 steps 17.0 and 26.0 (16 requests), 3 steps 23.1 and 26.8 (16), 26.5 and 28.8 (64), 4 steps 26.6 and 29.6; 6 steps
// 34.2 and 33.1 (16), 41.8 and 32.7 (64), 11 steps 60.5 and 53.1.  (Blocks of 12 tokens and 12 x 5 queries gain by parts
// up to 12 steps, 39.3 against 42.1, which this leaves.)
constexpr int kKv8Step = 128, kKv8Least = 2, kKv8Few = 4;
constexpr int kKv8Deal = (257 + 4) * 8 + (3 * 256 + 1) * 4;  // bytes of LDS

// References move by more than 2^kKv8Lazy only; P is at most 2^kKv8Lazy.  (BF16 terms have
// F32's range, so nothing is lost below.)
constexpr float kKv8Lazy = 8.0f;

// How queries of type QT and their probabilities enter the matrix cores.  (One term for BF16 queries'
// would add to a result's rounding to BF16, rms 1.7e-3, up to as much again: 2.7e-3 over few positions.)
template <class QT>
struct Kv8Kind;
template <>
struct Kv8Kind<float> {
    using T = _Float16;
    static constexpr int QTERMS = 2, PTERMS = 3;
};
template <>
struct Kv8Kind<_Float16> {
    using T = _Float16;
    static constexpr int QTERMS = 1, PTERMS = 2;
};
template <>
struct Kv8Kind<__bf16> {
    using T = __bf16;
    static constexpr int QTERMS = 1, PTERMS = 2;
};

template <class QT_, bool I8_, bool BLOCK8_, int D_, int RT_>
struct Kv8Cfg {
    using QT = QT_;
    using T = typename Kv8Kind<QT_>::T;
    static constexpr int QTERMS = Kv8Kind<QT_>::QTERMS, PTERMS = Kv8Kind<QT_>::PTERMS;
    static constexpr bool I8 = I8_, BLOCK8 = BLOCK8_;
    static constexpr int D = D_, RT = RT_, ROWS = 16 * RT_, KK = D_ / 32;
    // queries of more than 32 registers stay in LDS
    static constexpr bool QLDS = KK * RT * QTERMS > 8;
    static constexpr int QBYTES = RT * QTERMS * KK * 1024;
    static constexpr int LDS = 64 * D * 4 > QBYTES ? 64 * D * 4 : QBYTES;
    // after that: (M, l) of four waves' rows and the rows' factors; places of 32 positions of four waves
    static constexpr int PLACES = BLOCK8 ? 0 : 4 * 32 * (16 + 8);
    static constexpr int MORE = 1024 + PLACES;
    // Workgroups a CU: as many as spill nothing or little (F32 queries of 128 dimensions in three, 52 bytes
    // a lane: 16 requests 59.4 us, in two 53.5).
    static constexpr int WGS = D == 256 ? 1 : (D == 64 ? RT == 1 || (BLOCK8 && QTERMS == 1) : RT == 1 && BLOCK8 && QTERMS == 1) ? 3 : 2;
};

// Eight bytes as the operand of the score product.
template <bool I8>
__device__ __forceinline__ Vec8<_Float16>::type kv8_operand(uint32_t a, uint32_t b, _Float16) {
    union {
        f16x2 h[4];
        uint32_t w[4];
        Vec8<_Float16>::type v;
    } u;
    if (I8) {
        // 1024 + (x + 128) has x + 128 as F16's last bits
        a ^= 0x80808080u;
        b ^= 0x80808080u;
        u.w[0] = __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u);
        u.w[1] = __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u);
        u.w[2] = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);
        u.w[3] = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);
        const f16x2 less = {(_Float16)-1152.0f, (_Float16)-1152.0f};
#pragma unroll
        for (int i = 0; i < 4; ++i) u.h[i] += less;
    } else {
        u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
        u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
        u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
        u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    }
    return u.v;
}
// bytes `at` of a and b as a pair of BF16 (an int8's eight bits are BF16's upper half of F32)
__device__ __forceinline__ uint32_t kv8_pair(uint32_t a, uint32_t b, int at) {
    const float x = (float)(int8_t)(a >> (8 * at)), y = (float)(int8_t)(b >> (8 * at));
    return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
}
template <bool I8>
__device__ __forceinline__ Vec8<__bf16>::type kv8_operand(uint32_t a, uint32_t b, __bf16) {
    union {
        bf16x2 h[4];
        uint32_t w[4];
        Vec8<__bf16>::type v;
    } u;
    if (I8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t x = i < 2 ? a : b;
            const float lo = (float)(int8_t)(x >> (16 * (i & 1))), hi = (float)(int8_t)(x >> (16 * (i & 1) + 8));
            u.w[i] = __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
        }
    } else {
        u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
        u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
        u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
        u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
    }
    return u.v;
}
// Bytes 0..3 of eight positions' dwords as the operands of four output tiles.
template <bool I8>
__device__ __forceinline__ void kv8_values(const uint32_t (&x)[8], Vec8<__bf16>::type (&out)[4]) {
    union {
        bf16x2 h[4];
        uint32_t w[4];
        Vec8<__bf16>::type v;
    } u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = x[2 * i], b = x[2 * i + 1];
        if (I8) {
#pragma unroll
            for (int d = 0; d < 4; ++d) u[d].w[i] = kv8_pair(a, b, d);
        } else {
            const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05010400u), hi = __builtin_amdgcn_perm(b, a, 0x07030602u);
            u[0].h[i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
            u[1].h[i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
            u[2].h[i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
            u[3].h[i] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
        }
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) out[d] = u[d].v;
}

// Rows row0 .. row0 + 15 of the queries: of row n the dimensions (kk / 2) * 64 + g * 16 + (kk & 1) * 8 ..
// per lane, as the score product takes them.
template <class C>
struct Kv8Queries {
    using T = typename C::T;
    using QT = typename C::QT;
    static constexpr int KK = C::KK, N = 8 * sizeof(QT) / 16;
    union Piece {
        u32x4 v[N];
        QT e[8];
    } x[KK];

    __device__ __forceinline__ bool in(const AttnParams &p, const AttnSpan &s, int row0) const { return row0 + (int)(threadIdx.x & 15) < s.rows; }
    __device__ __forceinline__ int dim(int kk) const { return (kk >> 1) * 64 + ((threadIdx.x & 63) >> 4) * 16 + (kk & 1) * 8; }
    __device__ __forceinline__ void load(const AttnParams &p, const AttnSpan &s, int hk, int row0) {
        const int row = in(p, s, row0) ? row0 + (int)(threadIdx.x & 15) : 0;
        const int t = (int)fastdiv((uint32_t)row, p.group_div);
        const int h = hk * p.group + row - t * p.group;
        const QT *src = reinterpret_cast<const QT *>(p.q + (int64_t)(s.tok0 + t) * p.q_token + h * p.q_head);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            // (clamped, so that the loads need no branches)
            const QT *at = src + (dim(kk) < p.head_dim ? dim(kk) : 0);
            if (p.q_vec) {
#pragma unroll
                for (int i = 0; i < N; ++i) x[kk].v[i] = reinterpret_cast<const u32x4 *>(at)[i];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[kk].e[j] = at[j];
            }
        }
    }
    // to put(term, kk, vector); returns the row's factor c
    template <class PUT>
    __device__ __forceinline__ float give(const AttnParams &p, const AttnSpan &s, int row0, PUT put) const {
        const float sgn = p.scale < 0.0f ? -1.0f : 1.0f;
        const bool ok = in(p, s, row0);
        float top = 0.0f;
        auto value = [&](int kk, int j) { return ok && dim(kk) < p.head_dim ? (float)x[kk].e[j] * sgn : 0.0f; };
        float c = fabsf(p.scale) * kLog2e, f = 1.0f;
        if (C::QTERMS > 1) {
            // An F32 row of any magnitude: a power of two brings its largest value to 2^14..2^15, near the
            // end of F16's range.  The second term's smallest step, 2^-24, leaves each value its 22
            // bits down to 2^-17 of the row's largest (brought to 1..2, one at 2^-10 of it would keep 15).
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(value(kk, j)));
            top = xor_max(top);
            int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
            e = e > 127 ? 14 : e < -112 ? -112 : e;  // (not finite: as it is)
            f = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
            c *= __uint_as_float((uint32_t)(127 + e - 14) << 23);
        }
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            typename Vec8<T>::type v[C::QTERMS];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                T t8[C::QTERMS];
                split_terms<T, C::QTERMS>(value(kk, j) * f, t8);
#pragma unroll
                for (int i = 0; i < C::QTERMS; ++i) v[i][j] = t8[i];
            }
#pragma unroll
            for (int i = 0; i < C::QTERMS; ++i) put(i, kk, v[i]);
        }
        // (above zero, so that c * -inf of an unseen position stays -inf at a scale of 0)
        return fmaxf(c, 1e-37f);
    }
};

// Some byte of e4m3 that is NaN (0x7f, 0xff): zeroed, and told.
__device__ __forceinline__ bool kv8_nan(uint32_t &w) {
    const uint32_t m = w & 0x7f7f7f7fu, is = ((m + 0x01010101u) & 0x80808080u) >> 7;  // 1 in the bytes of NaN
    w &= ~(is * 255u);
    return is != 0;
}

// A row's reference in log2 units.
__device__ __forceinline__ float kv8_ref(float m, float c) { return m == -__builtin_inff() ? m : m * c; }

template <class C>
__device__ __forceinline__ void kv8_attn_item(const Kv8AttnParams &kp, const AttnSpan &s, int hk, int tile, char *lds) {
    using T = typename C::T;
    using QT = typename C::QT;
    using V8 = typename Vec8<T>::type;
    using B8 = Vec8<__bf16>::type;
    constexpr int D = C::D, RT = C::RT, KK = C::KK, QTERMS = C::QTERMS, PTERMS = C::PTERMS;
    constexpr int KJ = D / 64, VB = D / 16, VW = VB / 4;  // 16-byte pieces of a K row, bytes and dwords of a V piece
    const AttnParams &p = kp.a;
    const Kv8Cache &kv = kp.c;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (what follows from it is worked out for each item: kept from one to the next it spills)
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int row0 = tile * C::ROWS;
    const int least = attn_least<C::ROWS>(p, s, tile);
    char *more = lds + C::LDS;

    // this lane's pieces of a row (past the head: the first bytes again, for queries of 0 and outputs that are not stored)
    int kd[KJ];
#pragma unroll
    for (int j = 0; j < KJ; ++j) kd[j] = j * 64 + g * 16 < p.head_dim ? j * 64 + g * 16 : 0;
    const char *kb = kv.k + hk * kv.k_head, *vb = kv.v + hk * kv.v_head + (n * VB < p.head_dim ? n * VB : 0);
    const char *ksb = reinterpret_cast<const char *>(kv.k_scale) + hk * kv.s_head;
    const char *vsb = reinterpret_cast<const char *>(kv.v_scale) + hk * kv.s_head;

    u32x4 kf[2][KJ];
    uint32_t vf[8][VW];
    float ks[C::BLOCK8 ? 1 : 8], vs[C::BLOCK8 ? 1 : 8], vs_next[C::BLOCK8 ? 1 : 8];
    bool ok_next = false;      // this lane's positions (its first one) have a page
    uint32_t there_next = 0;   // without BLOCK8: bit r, position r of the step has one
    int page_k = 0, page_v = 0;
    int64_t v_at = 0;
    longlong2 *places = reinterpret_cast<longlong2 *>(more + 1024) + wave * 32;
    float2 *scales = reinterpret_cast<float2 *>(more + 1024 + 4 * 32 * 16) + wave * 32;
    // the page of position t (clamped to the span's last, so that nothing past a table is read)
    auto page_of = [&](int t) { return kv8_page(kv, (int)s.table_row, t < s.end ? t : s.end - 1); };
    auto slot_of = [&](int t) { return t - (int)(fastdiv((uint32_t)t, kv.page) * kv.page.d); };
    auto get_pages = [&](int t0) {
        if (C::BLOCK8) {
            page_k = page_of(t0 + (n >> 2) * 8);
            page_v = page_of(t0 + g * 8);
        } else {
            page_k = page_of(t0 + (lane & 31));
        }
    };
    auto load_k = [&](int t0) {
        if (C::BLOCK8) {
            const int tk = t0 + (n >> 2) * 8, tv = t0 + g * 8;
            const bool okk = tk < s.end && (uint32_t)page_k < (uint32_t)kv.n_pages;
            const bool okv = tv < s.end && (uint32_t)page_v < (uint32_t)kv.n_pages;
            const int64_t k_at = okk ? page_k * kv.k_page + slot_of(tk) * kv.k_token : 0;
            const int slot = okv ? slot_of(tv) : 0, pg = okv ? page_v : 0;
            v_at = pg * kv.v_page + slot * kv.v_token;
            const int64_t s_at = pg * kv.s_page + (int64_t)fastdiv((uint32_t)slot, kv.block) * kv.s_block;
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int j = 0; j < KJ; ++j)
                    kf[tt][j] = *reinterpret_cast<const u32x4 *>(kb + k_at + ((n & 3) + tt * 4) * kv.k_token + kd[j]);
            ks[0] = *reinterpret_cast<const float *>(ksb + s_at);
            vs_next[0] = *reinterpret_cast<const float *>(vsb + s_at);
            ok_next = okv;
        } else {
            const int t = t0 + (lane & 31);
            const bool ok = t < s.end && (uint32_t)page_k < (uint32_t)kv.n_pages;
            there_next = (uint32_t)__ballot(ok);
            const int pg = ok ? page_k : 0, slot = ok ? slot_of(t) : 0;
            const int64_t s_at = pg * kv.s_page + (int64_t)fastdiv((uint32_t)slot, kv.block) * kv.s_block;
            if (lane < 32) {
                places[lane] = make_longlong2(pg * kv.k_page + slot * kv.k_token, pg * kv.v_page + slot * kv.v_token);
                scales[lane] = make_float2(*reinterpret_cast<const float *>(ksb + s_at), *reinterpret_cast<const float *>(vsb + s_at));
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
                const int64_t at = places[(n >> 2) * 8 + tt * 4 + (n & 3)].x;
#pragma unroll
                for (int j = 0; j < KJ; ++j) kf[tt][j] = *reinterpret_cast<const u32x4 *>(kb + at + kd[j]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 x = scales[g * 8 + e];
                ks[C::BLOCK8 ? 0 : e] = x.x;
                vs_next[C::BLOCK8 ? 0 : e] = x.y;
            }
        }
    };
    auto load_v = [&]() {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const char *at = vb + (C::BLOCK8 ? v_at + e * kv.v_token : places[g * 8 + e].y);
            if constexpr (VW == 4) {
                const u32x4 x = *reinterpret_cast<const u32x4 *>(at);
#pragma unroll
                for (int w = 0; w < 4; ++w) vf[e][w] = x[w];
            } else if constexpr (VW == 2) {
                const uint2 x = *reinterpret_cast<const uint2 *>(at);
                vf[e][0] = x.x;
                vf[e][1] = x.y;
            } else {
                vf[e][0] = *reinterpret_cast<const uint32_t *>(at);
            }
        }
    };
    // the queries, one row tile per wave, then the first positions
    Kv8Queries<C> own;
    if (wave < RT) own.load(p, s, hk, row0 + wave * 16);
    int t0 = s.beg + wave * 32;
    if (t0 < s.end) {
        get_pages(t0);
        load_k(t0);
        load_v();
        get_pages(t0 + 128);
    }
    __syncthreads();  // (LDS may still be read for the item before)
    AttnRows<RT, D> w;
    attn_rows<RT, D>(p, s, row0, w);
    V8 q[C::QLDS ? 1 : RT][QTERMS][KK];
    float *cs = reinterpret_cast<float *>(more);
    if (wave < RT) {
        const float c = own.give(p, s, row0 + wave * 16, [&](int i, int kk, V8 v) {
            *reinterpret_cast<V8 *>(lds + ((wave * QTERMS + i) * KK + kk) * 1024 + lane * 16) = v;
        });
        if (g == 0) cs[wave * 16 + n] = c;
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        w.c[rt] = cs[rt * 16 + n];
        w.ref[rt] = 0.0f;
    }
    if (!C::QLDS) {
#pragma unroll
        for (int f = 0; f < RT * QTERMS * KK; ++f)
            q[C::QLDS ? 0 : f / (QTERMS * KK)][f / KK % QTERMS][f % KK] = *reinterpret_cast<const V8 *>(lds + f * 1024 + lane * 16);
    }
    bool fine = true;  // of the values at and after the first step that ends past `least`
    for (; t0 < s.end; t0 += 128) {
        const bool ok = ok_next;
        const uint32_t there = there_next;
        // positions that some row does not see, or that are not there
        const bool differ = t0 + 32 > least, careful = differ || (C::BLOCK8 ? !__all(ok) : there != 0xffffffffu);
#pragma unroll
        for (int e = 0; e < (C::BLOCK8 ? 1 : 8); ++e) vs[e] = vs_next[e];
        f32x4 sx[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sx[rt][0] = sx[rt][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            V8 ka[2];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) ka[tt] = kv8_operand<C::I8>(kf[tt][kk >> 1][(kk & 1) * 2], kf[tt][kk >> 1][(kk & 1) * 2 + 1], T());
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int i = 0; i < QTERMS; ++i) {
                    const V8 qv = C::QLDS ? *reinterpret_cast<const V8 *>(lds + ((rt * QTERMS + i) * KK + kk) * 1024 + lane * 16)
                                          : q[C::QLDS ? 0 : rt][i][kk];
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt) sx[rt][tt] = mfma(ka[tt], qv, sx[rt][tt]);
                }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int e = 0; e < 8; ++e) sx[rt][e >> 2][e & 3] *= ks[C::BLOCK8 ? 0 : e];
        // The next step's K leaves before this one's softmax (past the end: the first bytes of the cache)
        load_k(t0 + 128);
        get_pages(t0 + 256);
        if (careful) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int u = g * 8 + e;
                const bool here = C::BLOCK8 ? ok && t0 + u < s.end : (there >> u) & 1;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    if (!here || t0 + u >= w.limit[rt]) sx[rt][e >> 2][e & 3] = -__builtin_inff();
                if (!C::I8) {
#pragma unroll
                    for (int x = 0; x < VW; ++x)
                        if (!here) vf[e][x] = 0;
                }
            }
        }
        // (where rows see the same, the products take what is there to all of them)
        if (!C::I8 && differ) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int x = 0; x < VW; ++x) fine = !kv8_nan(vf[e][x]) && fine;
        }
        // new references when some row passes its old one by 2^kKv8Lazy (-inf: always)
        float top[RT];
        bool over = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            top[rt] = fmaxf(fmaxf(sx[rt][0][0], sx[rt][0][1]), sx[rt][0][2]);
            top[rt] = fmaxf(fmaxf(top[rt], sx[rt][0][3]), sx[rt][1][0]);
            top[rt] = fmaxf(fmaxf(top[rt], sx[rt][1][1]), sx[rt][1][2]);
            top[rt] = fmaxf(top[rt], sx[rt][1][3]);
            over |= top[rt] > w.over[rt];
        }
        if (__any(over)) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float mn = fmaxf(w.m[rt], xor_max(top[rt]));
                // (nothing was summed yet, or nothing changes: also keeps inf - inf and 0 * inf out)
                const float f = w.m[rt] == -__builtin_inff() || w.m[rt] == mn ? 1.0f : __builtin_amdgcn_exp2f((w.m[rt] - mn) * w.c[rt]);
                w.m[rt] = mn;
                w.over[rt] = mn + kKv8Lazy / w.c[rt];
                w.ref[rt] = mn == -__builtin_inff() ? 0.0f : -mn * w.c[rt];
                w.l[rt] *= f;
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt) w.o[rt][dt] *= f;
            }
        }
        B8 pf[RT][PTERMS];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sx[rt][e >> 2][e & 3], w.c[rt], w.ref[rt]));
                w.l[rt] += x;
                // (a scale that is not finite stays with the rows that see it)
                float y = x * vs[C::BLOCK8 ? 0 : e];
                if (careful) y = x == 0.0f ? 0.0f : y;
                __bf16 t8[PTERMS];
                split_terms<__bf16, PTERMS>(y, t8);
#pragma unroll
                for (int i = 0; i < PTERMS; ++i) pf[rt][i][e] = t8[i];
            }
#pragma unroll
        for (int x = 0; x < VW; ++x) {
            uint32_t col[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) col[e] = vf[e][x];
            B8 va[4];
            kv8_values<C::I8>(col, va);
#pragma unroll
            for (int d = 0; d < 4; ++d)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int i = 0; i < PTERMS; ++i) w.o[rt][x * 4 + d] = mfma(va[d], pf[rt][i], w.o[rt][x * 4 + d]);
        }
        load_v();
    }
    if (!C::I8 && !__all(fine)) {
        // bytes of NaN where rows see different positions: to the rows that see them
        for (t0 = s.beg + wave * 32; t0 < s.end; t0 += 128)
            for (int t = t0; t0 + 32 > least && t < t0 + 32 && t < s.end; ++t) {
                const int page = page_of(t);
                if ((uint32_t)page >= (uint32_t)kv.n_pages) continue;
                const uint8_t *v = reinterpret_cast<const uint8_t *>(kv.v + hk * kv.v_head + page * kv.v_page + slot_of(t) * kv.v_token);
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int dt = 0; dt < VB; ++dt) {
                        const int d = (g * 4 + j) * VB + dt;
                        if (d >= p.head_dim || (v[d] & 0x7f) != 0x7f) continue;
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
                            if (t < w.limit[rt]) w.o[rt][dt][j] = __builtin_nanf("");
                    }
            }
    }

    // the four waves' parts of each row tile join in LDS
    float *ol = reinterpret_cast<float *>(lds);      // [wave][16][D], pieces of four dimensions xored with the row
    float2 *ml = reinterpret_cast<float2 *>(more);   // [wave][16]
    constexpr int Q4 = D / 4;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = xor_sum(w.l[rt]);
        const int left = s.rows - row0 - rt * 16, rows = left < 16 ? left : 16;
        __syncthreads();
        if (n < rows) {
            if (g == 0) ml[wave * 16 + n] = make_float2(kv8_ref(w.m[rt], w.c[rt]), sum);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int x = 0; x < VW; ++x) {
                    f32x4 y;
#pragma unroll
                    for (int d = 0; d < 4; ++d) y[d] = w.o[rt][x * 4 + d][j];
                    *reinterpret_cast<f32x4 *>(ol + (wave * 16 + n) * D + ((((g * 4 + j) * VW + x) ^ n) * 4)) = y;
                }
        }
        __syncthreads();
        for (int x = tid; x < rows * Q4; x += 256) {
            const int r = x / Q4, d4 = x % Q4;
            float M = -__builtin_inff();
#pragma unroll
            for (int v = 0; v < 4; ++v) M = fmaxf(M, ml[v * 16 + r].x);
            f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
            float ls = 0.0f;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float2 e = ml[v * 16 + r];
                if (e.y == 0.0f) continue;  // the row sees nothing of this wave's part
                const float f = __builtin_amdgcn_exp2f(e.x == M ? 0.0f : e.x - M);
                ls += e.y * f;
                acc += *reinterpret_cast<const f32x4 *>(ol + (v * 16 + r) * D + ((d4 ^ r) * 4)) * f;
            }
            if (s.slot < 0) {
                attn_emit<QT>(p, s, hk, row0 + rt * 16 + r, d4 * 4, acc, M, ls);
            } else if (d4 * 4 < p.head_dim) {
                const int64_t at = (int64_t)s.slot * C::ROWS + rt * 16 + r;
                if (d4 == 0) p.part_ml[at] = make_float2(M, ls);
                *reinterpret_cast<f32x4 *>(p.part_o + at * p.head_dim + d4 * 4) = acc;
            }
        }
    }
}

// What request r takes: its rows, tiles of them and steps.
template <int TILE_ROWS>
struct Kv8Request {
    int t0, t1, len;
    __device__ __forceinline__ Kv8Request(int first, int end, int n) : t0(first), t1(end), len(n) {}
    __device__ __forceinline__ Kv8Request(const AttnParams &p, int r) {
        attn_tokens(p, r, t0, t1);
        len = attn_suffix(p, r);
    }
    __device__ __forceinline__ int rows(const AttnParams &p) const { return (t1 - t0) * p.group; }
    __device__ __forceinline__ int tiles(const AttnParams &p) const { return (rows(p) + TILE_ROWS - 1) / TILE_ROWS; }
    __device__ __forceinline__ int steps() const { return (len + kKv8Step - 1) / kKv8Step; }
    // (below 2^31)
    __device__ __forceinline__ int all(const AttnParams &p) const { return steps() * tiles(p) * p.n_head_kv; }
};
// Steps are counted in whole numbers below 2^53, held in 64-bit floats: quotients are 15 instructions
// instead of 150, and exact once rounded down.
__device__ __forceinline__ double kv8_quotient(double x, double y) { return floor(x / y); }
// Steps `step` and up of a request, n of them at most, whose partial results go to `slot` unless these
// are all.
template <int TILE_ROWS>
__device__ __forceinline__ AttnSpan kv8_span(const AttnParams &p, const Kv8Request<TILE_ROWS> &q, int r, int step, int n, int slot) {
    AttnSpan s;
    s.beg = step * kKv8Step;
    s.end = n < q.steps() - step ? s.beg + n * kKv8Step : q.len;
    s.rows = q.rows(p);
    s.tok0 = q.t0;
    s.causal = q.len - (q.t1 - q.t0);
    s.table_row = r;
    s.slot = step == 0 && n >= q.steps() ? -1 : slot;
    return s;
}
// steps of a share, of all steps
__device__ __forceinline__ double kv8_share(const Kv8AttnParams &kp, double all) {
    return fmax(kv8_quotient(all + (kp.shares - 1), kp.shares), kKv8Least);
}

// Parts of one length, where they are of a few steps; else all steps of all requests, KV heads and
// tiles, in that order, dealt out evenly to as many workgroups as the card holds at once, whatever
// the requests' lengths.  Tiles of several parts are joined by a kernel of its own.  (64 requests of
// 512 to 8192 positions: 232 us with two parts of one length a request, 183 with eight, 151 dealt out;
// 12 x 5 F16 tokens over up to 3001 positions: 16.2 us with parts of three steps, 21.7 dealt out, which
// has to count all lengths first, and to wait for a second tile's first positions.)
// (two kernels: in one, each keeps the other's arguments in registers)
template <class C>
__global__ __launch_bounds__(256, C::WGS) void kv8_attn_kernel(Kv8AttnParams kp) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const AttnParams &p = kp.a;
    // part (slowest), request, KV head, tile
    const int item = xcd_item(blockIdx.x, p.suf_items);
    int x = item / p.suf_tiles;
    const int tile = item - x * p.suf_tiles, hk = x % p.n_head_kv;
    x /= p.n_head_kv;
    const int r = x % p.n_requests, step = x / p.n_requests * kp.each;
    const Kv8Request<C::ROWS> q(p, r);
    // (the first part of a request that sees nothing writes its empty rows)
    if (tile >= q.tiles(p) || (step > 0 && step >= q.steps())) return;
    kv8_attn_item<C>(kp, kv8_span(p, q, r, step, kp.each, item), hk, tile, lds);
}

template <class C>
__global__ __launch_bounds__(256, C::WGS) void kv8_attn_dealt_kernel(Kv8AttnParams kp) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const AttnParams &p = kp.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    using Request = Kv8Request<C::ROWS>;
    // 256 requests: where they begin in steps, and the last one ends; what they take
    double *begins = reinterpret_cast<double *>(lds + C::LDS + C::MORE), *sums = begins + 257;
    int *tokens = reinterpret_cast<int *>(sums + 4), *ends = tokens + 256, *lens = ends + 256, &found = lens[256];
    // requests r0 .. r0 + 255, whose steps begin at `from`: returns where they end
    auto number = [&](int r0, double from) {
        Request q(0, 0, 0);
        if (r0 + tid < p.n_requests) q = Request(p, r0 + tid);
        const double own = q.all(p), inc = wave_scan(own);
        __syncthreads();
        tokens[tid] = q.t0;
        ends[tid] = q.t1;
        lens[tid] = q.len;
        if (lane == 63) sums[wave] = inc;
        __syncthreads();
        double all = from;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i == wave) begins[tid] = all + inc - own;
            all += sums[i];
        }
        if (tid == 0) begins[256] = all;
        __syncthreads();
        return lane_of(all, 0);
    };
    const int share = xcd_item(blockIdx.x, kp.shares);
    double total = 0;
    int r0 = 0;
    for (; r0 < p.n_requests; r0 += 256) {
        total = number(r0, total);
        if (share == 0 && r0 + tid < p.n_requests) kp.starts[r0 + tid] = begins[tid];
    }
    if (share == 0 && tid == 0) kp.starts[p.n_requests] = total;
    const double each = kv8_share(kp, total);
    const double first = lane_of(share * each, 0), last = lane_of(fmin(first + each, total), 0);
    if (first >= last) return;
    // (the last 256 requests' numbers are there; the first ones again where there are more)
    r0 -= 256;
    if (r0 > 0) {
        r0 = 0;
        number(0, 0);
    }
    for (double at = first; at < last;) {
        while (at >= lane_of(begins[256], 0)) {
            r0 += 256;
            number(r0, lane_of(begins[256], 0));
        }
        if (begins[tid] <= at && at < begins[tid + 1]) found = tid;
        __syncthreads();
        const int in = __builtin_amdgcn_readfirstlane(found);
        const Request q(__builtin_amdgcn_readfirstlane(tokens[in]), __builtin_amdgcn_readfirstlane(ends[in]), __builtin_amdgcn_readfirstlane(lens[in]));
        const int past = (int)(at - lane_of(begins[in], 0));
        const int which = past / q.steps(), step = past - which * q.steps();
        const int hk = which / q.tiles(p), tile = which - hk * q.tiles(p);
        const int n = (int)fmin(last - at, q.steps() - step);
        kv8_attn_item<C>(kp, kv8_span(p, q, r0 + in, step, n, 2 * share + (at > first)), hk, tile, lds);
        at += n;
    }
}

// Joins the parts of the tiles that several workgroups had: join_groups threads for each four
// dimensions of a row.
template <class QT, int TILE_ROWS>
__global__ __launch_bounds__(kJoinThreads) void kv8_join_kernel(Kv8AttnParams kp) {
    __shared__ f32x4 acc[kJoinThreads];
    __shared__ float2 mls[kJoinThreads];
    const AttnParams &p = kp.a;
    const JoinThread me(threadIdx.x, p.head_dim, p.join_groups, p.join_rows);
    const int d4 = me.d4, sub = me.sub;
    const int64_t item = (int64_t)blockIdx.x * p.join_rows + me.which;
    const int64_t rt = item / p.n_head;
    const int head = (int)(item - rt * p.n_head);
    const int64_t r = rt / p.n_q;
    const int t = (int)(rt - r * p.n_q);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f, M = -__builtin_inff();
    // A part in which the row sees nothing (l of 0) adds nothing, whatever its values.
    auto add = [&](float2 e, f32x4 x) {
        if (e.y == 0.0f) return;
        const float mn = fmaxf(M, e.x);
        const float f = M == mn || l == 0.0f ? 1.0f : __builtin_amdgcn_exp2f(M - mn);
        const float g = e.x == mn ? 1.0f : __builtin_amdgcn_exp2f(e.x - mn);
        l = l * f + e.y * g;
        o = o * f + x * g;
        M = mn;
    };
    int64_t tok = -1;
    if (me.there && r < p.n_requests) {
        const Kv8Request<TILE_ROWS> q(p, (int)r);
        const int hk = head / p.group, row = t * p.group + head - hk * p.group, tile = row / TILE_ROWS;
        if (row < q.rows(p)) {
            // the number of parts, and where they are; none to join where one workgroup had all
            int parts, first = 0;
            int64_t slot0, stride;
            if (kp.shares) {
                const double each = kv8_share(kp, kp.starts[p.n_requests]);
                const double beg = kp.starts[r] + (double)((hk * q.tiles(p) + tile) * q.steps());
                const int b0 = (int)kv8_quotient(beg, each);
                parts = q.len ? (int)kv8_quotient(beg + (q.steps() - 1), each) - b0 + 1 : 0;
                first = beg > b0 * each;
                slot0 = 2 * (int64_t)b0;
                stride = 2;
            } else {
                parts = (q.steps() + kp.each - 1) / kp.each;
                stride = (int64_t)p.n_requests * p.n_head_kv * p.suf_tiles;
                slot0 = (r * p.n_head_kv + hk) * p.suf_tiles + tile;
            }
            // (a request of no positions was dealt out to nobody)
            if (parts > 1 || (parts == 0 && kp.shares)) tok = q.t0 + t;
            if (parts <= 1) parts = 0;
            constexpr int U = 4;
            for (int i0 = sub; i0 < parts; i0 += p.join_groups * U) {
                float2 e[U];
                f32x4 x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = i0 + u * p.join_groups < parts ? i0 + u * p.join_groups : i0;
                    const int64_t slot = slot0 + i * stride + (i == 0 ? first : 0), at = slot * TILE_ROWS + row - tile * TILE_ROWS;
                    e[u] = p.part_ml[at];
                    x[u] = *reinterpret_cast<const f32x4 *>(p.part_o + at * p.head_dim + d4 * 4);
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i0 + u * p.join_groups < parts) add(e[u], x[u]);
            }
        }
    }
    if (p.join_groups > 1) {
        acc[threadIdx.x] = o;
        mls[threadIdx.x] = make_float2(M, l);
        __syncthreads();
        if (me.collects())
            for (int i = 1; i < p.join_groups; ++i) {
                const int at = JoinThread::place(threadIdx.x, p.head_dim, i);
                add(mls[at], acc[at]);
            }
    }
    if (tok < 0 || !me.collects()) return;
    QT *dst = reinterpret_cast<QT *>(p.dst + tok * p.dst_token + head * p.dst_head) + d4 * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) dst[j] = (QT)(l == 0.0f ? 0.0f : o[j] / l);
    if (d4 == 0 && p.lse) p.lse[tok * p.n_head + head] = l == 0.0f ? -__builtin_inff() : (M + log2f(l)) * kLn2;
}

struct Kv8AttnPlan {
    Kv8AttnParams p;
    int dim, rt;  // padded head dimension, row tiles
    bool i8, block8;
    size_t bytes, start_bytes;
    int64_t slots;  // of parts that are joined
    int lds, wgs;  // wgs: workgroups a CU
    const void *kernel, *dealt, *join;
};
// (an instantiation per type of the queries, each in a file of its own)
void kv8_attn_f32(Kv8AttnPlan &pl);
void kv8_attn_f16(Kv8AttnPlan &pl);
void kv8_attn_bf16(Kv8AttnPlan &pl);

template <class C>
void kv8_attn_instance(Kv8AttnPlan &pl) {
    pl.kernel = reinterpret_cast<const void *>(&kv8_attn_kernel<C>);
    pl.dealt = reinterpret_cast<const void *>(&kv8_attn_dealt_kernel<C>);
    pl.join = reinterpret_cast<const void *>(&kv8_join_kernel<typename C::QT, C::ROWS>);
    pl.lds = C::LDS + C::MORE;
    pl.wgs = C::WGS;
}
template <class QT, bool I8, bool BLOCK8>
void kv8_attn_kernel_of(Kv8AttnPlan &pl) {
    if (pl.dim == 64) pl.rt == 1 ? kv8_attn_instance<Kv8Cfg<QT, I8, BLOCK8, 64, 1>>(pl) : kv8_attn_instance<Kv8Cfg<QT, I8, BLOCK8, 64, 2>>(pl);
    else if (pl.dim == 128) pl.rt == 1 ? kv8_attn_instance<Kv8Cfg<QT, I8, BLOCK8, 128, 1>>(pl) : kv8_attn_instance<Kv8Cfg<QT, I8, BLOCK8, 128, 2>>(pl);
    else kv8_attn_instance<Kv8Cfg<QT, I8, BLOCK8, 256, 1>>(pl);
}
template <class QT>
void kv8_attn_kernel_of(Kv8AttnPlan &pl) {
    if (pl.i8) pl.block8 ? kv8_attn_kernel_of<QT, true, true>(pl) : kv8_attn_kernel_of<QT, true, false>(pl);
    else pl.block8 ? kv8_attn_kernel_of<QT, false, true>(pl) : kv8_attn_kernel_of<QT, false, false>(pl);
}

}  // namespace q4k

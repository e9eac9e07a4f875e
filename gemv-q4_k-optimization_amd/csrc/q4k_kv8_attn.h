// q4k_kv8_attn.h -- the attention kernel over paged caches of 8 bits
// (q4k_kv8_attn.hip).
//
// A workgroup takes up to 16 * RT query rows (token, head of the group) of one
// request and KV head and a stretch of its positions; its four waves go over steps
// of 32 positions of their own, once, with a running maximum and sum, and join at
// the end:
//   S^T = (K Q^T) ks      v_mfma_f32_16x16x32 on the bytes as F16 (BF16), exact
//   P = exp2(c S - M)     in the lanes that hold S
//   O^T += V^T (P vs)^T   v_mfma_f32_16x16x32_bf16, P vs as 1 to 3 BF16 terms
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
#pragma once

#include "q4k_attn.h"
#include "q4k_kv8.h"

namespace q4k {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct Kv8AttnParams {
    AttnParams a;  // rows and partial results; `suf` parts only, no AttnCache
    Kv8Cache c;
    // Where the positions are dealt out: workgroups that share them (else 0), the number of steps
    // before each request's and, last, of all, for the join.  (a.join stays 0: attn_emit writes dst.)
    int shares;
    int64_t *starts;
};

// Positions of a step of four waves; the least steps a workgroup takes (12 x 5 F16 tokens over 3001
// positions: 1 step @@, 2 @@, 4 @@ us).
constexpr int kKv8Step = 128, kKv8Least = 2;
constexpr int kKv8Deal = (257 + 4 + 1) * 8;  // bytes of LDS

// References move by more than 2^kKv8Lazy only; P is at most 2^kKv8Lazy.  (BF16 terms have
// F32's range, so nothing is lost below.)
constexpr float kKv8Lazy = 8.0f;

// How queries of type QT and their probabilities enter the matrix cores.
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
    static constexpr int QTERMS = 1, PTERMS = 1;
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
    static constexpr int WGS = D == 256 ? 1 : D == 128 && RT == 2 ? 2 : 3;  // workgroups a CU
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

// Rows row0 .. row0 + 15: of row n the dimensions (kk / 2) * 64 + g * 16 + (kk & 1) * 8 ..
// per lane, as the score product takes them, handed to put(term, kk, vector).
// Returns the row's factor c.
template <class C, class PUT>
__device__ __forceinline__ float kv8_queries(const AttnParams &p, const AttnSpan &s, int hk, int row0, PUT put) {
    using T = typename C::T;
    using QT = typename C::QT;
    using V8 = typename Vec8<T>::type;
    constexpr int KK = C::KK;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const float sgn = p.scale < 0.0f ? -1.0f : 1.0f;
    const int row = row0 + n;
    const bool ok = row < s.rows;
    const int t = (int)fastdiv((uint32_t)(ok ? row : 0), p.group_div);
    const int h = hk * p.group + (ok ? row : 0) - t * p.group;
    const QT *src = reinterpret_cast<const QT *>(p.q + (int64_t)(s.tok0 + t) * p.q_token + h * p.q_head);
    float x[KK][8];
    float top = 0.0f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
        // (clamped, so that the loads need no branches)
        const int d = (kk >> 1) * 64 + g * 16 + (kk & 1) * 8;
        const bool in = ok && d < p.head_dim;
        const QT *at = src + (d < p.head_dim ? d : 0);
        if (p.q_vec) {
            constexpr int N = 8 * sizeof(QT) / 16;
            union {
                u32x4 v[N];
                QT e[8];
            } u;
#pragma unroll
            for (int i = 0; i < N; ++i) u.v[i] = reinterpret_cast<const u32x4 *>(at)[i];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[kk][j] = (float)u.e[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[kk][j] = (float)at[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[kk][j] = in ? x[kk][j] * sgn : 0.0f;
            top = fmaxf(top, fabsf(x[kk][j]));
        }
    }
    float c = fabsf(p.scale) * kLog2e, f = 1.0f;
    if (C::QTERMS > 1) {
        // an F32 row of any magnitude: a power of two brings its largest value to 1..2
        top = xor_max(top);
        int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
        e = e < -126 || e > 127 ? 0 : e > 126 ? 126 : e;
        f = __uint_as_float((uint32_t)(127 - e) << 23);
        c *= __uint_as_float((uint32_t)(127 + e) << 23);
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
        V8 v[C::QTERMS];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            T t8[C::QTERMS];
            split_terms<T, C::QTERMS>(x[kk][j] * f, t8);
#pragma unroll
            for (int i = 0; i < C::QTERMS; ++i) v[i][j] = t8[i];
        }
#pragma unroll
        for (int i = 0; i < C::QTERMS; ++i) put(i, kk, v[i]);
    }
    // (above zero, so that c * -inf of an unseen position stays -inf at a scale of 0)
    return fmaxf(c, 1e-37f);
}

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
    int t0 = s.beg + wave * 32;
    if (t0 < s.end) {
        get_pages(t0);
        load_k(t0);
        load_v();
        get_pages(t0 + 128);
    }
    __syncthreads();  // (LDS may still be read for the item before)
    // the queries, one row tile per wave, while the first positions are on their way
    AttnRows<RT, D> w;
    attn_rows<RT, D>(p, s, row0, w);
    V8 q[C::QLDS ? 1 : RT][QTERMS][KK];
    float *cs = reinterpret_cast<float *>(more);
    if (wave < RT) {
        const float c = kv8_queries<C>(p, s, hk, row0 + wave * 16, [&](int i, int kk, V8 v) {
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
        const bool careful = t0 + 32 > least || (C::BLOCK8 ? !__all(ok) : there != 0xffffffffu);
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
                    for (int x = 0; x < VW; ++x) {
                        if (!here) vf[e][x] = 0;
                        fine = !kv8_nan(vf[e][x]) && fine;
                    }
                }
            }
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
        __syncthreads();
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
        __syncthreads();
        for (int x = tid; x < 16 * Q4; x += 256) {
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
            } else if (row0 + rt * 16 + r < s.rows && d4 * 4 < p.head_dim) {
                const int64_t at = (int64_t)s.slot * C::ROWS + rt * 16 + r;
                if (d4 == 0) p.part_ml[at] = make_float2(M, ls);
                *reinterpret_cast<f32x4 *>(p.part_o + at * p.head_dim + d4 * 4) = acc;
            }
        }
    }
}

// What request r takes: its rows, tiles of them and steps.
struct Kv8Request {
    int t0, rows, tiles, len, steps;
    __device__ __forceinline__ Kv8Request(const AttnParams &p, int r, int tile_rows) {
        int t1;
        attn_tokens(p, r, t0, t1);
        rows = (t1 - t0) * p.group;
        tiles = (rows + tile_rows - 1) / tile_rows;
        len = attn_suffix(p, r);
        steps = (len + kKv8Step - 1) / kKv8Step;
    }
    __device__ __forceinline__ long long all(const AttnParams &p) const { return (long long)steps * tiles * p.n_head_kv; }
};
__device__ __forceinline__ long long kv8_uniform(long long x) {
    const unsigned lo = __builtin_amdgcn_readfirstlane((int)x), hi = __builtin_amdgcn_readfirstlane((int)(x >> 32));
    return (long long)((unsigned long long)hi << 32 | lo);
}
// steps of a share, of all steps
__device__ __forceinline__ long long kv8_share(const Kv8AttnParams &kp, long long all) {
    const long long x = (all + kp.shares - 1) / kp.shares;
    return x < kKv8Least ? kKv8Least : x;
}
__device__ __forceinline__ long long kv8_wave_scan(long long x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const long long y = __shfl_up(x, d);
        x += lane >= d ? y : 0;
    }
    return x;
}

// Short caches: a workgroup for each tile of rows.  Longer ones: all steps of all requests, KV heads
// and tiles, in that order, are dealt out evenly to as many workgroups as the card holds at
// once, whatever the requests' lengths; a tile that more than one of them works on is joined by a
// kernel of its own.  (64 requests of 512 to 8192 positions: 232 us with splits of one length for all,
// two a request; 183 with eight; @@ dealt out.)
template <class C>
__global__ __launch_bounds__(256, C::WGS) void kv8_attn_kernel(Kv8AttnParams kp) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const AttnParams &p = kp.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // where 256 requests begin and the last one ends, in steps; sums of the waves'; the request in turn
    long long *begins = reinterpret_cast<long long *>(lds + C::LDS + C::MORE), *sums = begins + 257;
    int &found = *reinterpret_cast<int *>(sums + 4);
    // requests r0 .. r0 + 255, whose steps begin at `from`: returns where they end
    auto number = [&](int r0, long long from) {
        const long long own = r0 + tid < p.n_requests ? Kv8Request(p, r0 + tid, C::ROWS).all(p) : 0;
        const long long inc = kv8_wave_scan(own);
        __syncthreads();
        if (lane == 63) sums[wave] = inc;
        __syncthreads();
        long long all = from;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i == wave) begins[tid] = all + inc - own;
            all += sums[i];
        }
        if (tid == 0) begins[256] = all;
        __syncthreads();
        return kv8_uniform(all);
    };
    const int share = kp.shares ? xcd_item(blockIdx.x, kp.shares) : 0;
    long long at = 0, last = 0;
    int r0 = 0;
    if (kp.shares) {
        long long total = 0;
        for (; r0 < p.n_requests; r0 += 256) {
            const long long from = total;
            total = number(r0, from);
            if (share == 0 && r0 + tid < p.n_requests) kp.starts[r0 + tid] = begins[tid];
        }
        if (share == 0 && tid == 0) kp.starts[p.n_requests] = total;
        const long long each = kv8_share(kp, total);
        at = share * each;
        last = at + each < total ? at + each : total;
        if (at >= last) return;
        // (the last 256 requests' numbers are there; the first ones again where there are more)
        r0 -= 256;
        if (r0 > 0) {
            r0 = 0;
            number(0, 0);
        }
    }
    const long long first = at;
    do {
        int r, hk, tile, step = 0, n;
        if (kp.shares) {
            while (at >= kv8_uniform(begins[256])) {
                r0 += 256;
                number(r0, kv8_uniform(begins[256]));
            }
            if (begins[tid] <= at && at < begins[tid + 1]) found = tid;
            __syncthreads();
            const int in = __builtin_amdgcn_readfirstlane(found);
            r = r0 + in;
            const Kv8Request q(p, r, C::ROWS);
            const int past = (int)(at - kv8_uniform(begins[in]));  // (a request's steps are below 2^31)
            const int which = past / q.steps;
            step = past - which * q.steps;
            hk = which / q.tiles;
            tile = which - hk * q.tiles;
            n = last - at < q.steps - step ? (int)(last - at) : q.steps - step;
        } else {
            const int item = xcd_item(blockIdx.x, p.suf_items), x = item / p.suf_tiles;
            tile = item - x * p.suf_tiles;
            r = x / p.n_head_kv;
            hk = x - r * p.n_head_kv;
            n = kKv8Least;
        }
        const Kv8Request q(p, r, C::ROWS);
        AttnSpan s;
        s.beg = step * kKv8Step;
        s.end = n < q.steps - step ? s.beg + n * kKv8Step : q.len;
        s.rows = q.rows;
        s.tok0 = q.t0;
        s.causal = q.len - q.rows / p.group;
        s.table_row = r;
        s.slot = !kp.shares || n == q.steps ? -1 : 2 * share + (at > first);
        if (tile < q.tiles) kv8_attn_item<C>(kp, s, hk, tile, lds);
        at += n;
    } while (at < last);
}

// Joins the parts of the tiles that several workgroups had: join_groups threads for each four
// dimensions of a row.
template <class QT, int TILE_ROWS>
__global__ __launch_bounds__(256) void kv8_join_kernel(Kv8AttnParams kp) {
    __shared__ f32x4 acc[256];
    __shared__ float2 mls[256];
    const AttnParams &p = kp.a;
    const int q4 = p.head_dim / 4;
    const int grp = threadIdx.x / q4, d4 = threadIdx.x - grp * q4;
    const int sub = grp % p.join_groups, which = grp / p.join_groups;
    const int64_t item = (int64_t)blockIdx.x * p.join_rows + which;
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
    if (which < p.join_rows && r < p.n_requests) {
        const Kv8Request q(p, (int)r, TILE_ROWS);
        const int hk = head / p.group, row = t * p.group + head - hk * p.group, tile = row / TILE_ROWS;
        if (row < q.rows) {
            const long long each = kv8_share(kp, kp.starts[p.n_requests]);
            const long long beg = kp.starts[r] + ((long long)hk * q.tiles + tile) * q.steps;
            const int b0 = (int)(beg / each), b1 = q.steps ? (int)((beg + q.steps - 1) / each) : b0;
            // (one workgroup's own rows are where they belong; a row of no positions is nobody's)
            if (b1 > b0 || q.steps == 0) tok = q.t0 + t;
            constexpr int U = 4;
            for (int i0 = sub; b1 > b0 && i0 <= b1 - b0; i0 += p.join_groups * U) {
                float2 e[U];
                f32x4 x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = i0 + u * p.join_groups <= b1 - b0 ? i0 + u * p.join_groups : i0;
                    const int64_t slot = 2 * (int64_t)(b0 + i) + (i == 0 && beg > b0 * each), at = slot * TILE_ROWS + row - tile * TILE_ROWS;
                    e[u] = p.part_ml[at];
                    x[u] = *reinterpret_cast<const f32x4 *>(p.part_o + at * p.head_dim + d4 * 4);
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (i0 + u * p.join_groups <= b1 - b0) add(e[u], x[u]);
            }
        }
    }
    if (p.join_groups > 1) {
        acc[threadIdx.x] = o;
        mls[threadIdx.x] = make_float2(M, l);
        __syncthreads();
        if (sub == 0)
            for (int i = 1; i < p.join_groups; ++i) add(mls[threadIdx.x + i * q4], acc[threadIdx.x + i * q4]);
    }
    if (tok < 0 || sub != 0) return;
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
    int lds, wgs;  // wgs: workgroups a CU
    const void *kernel, *join;
};
// (an instantiation per type of the queries, each in a file of its own)
void kv8_attn_f32(Kv8AttnPlan &pl);
void kv8_attn_f16(Kv8AttnPlan &pl);
void kv8_attn_bf16(Kv8AttnPlan &pl);

template <class C>
void kv8_attn_instance(Kv8AttnPlan &pl) {
    pl.kernel = reinterpret_cast<const void *>(&kv8_attn_kernel<C>);
    pl.join = reinterpret_cast<const void *>(&kv8_join_kernel<typename C::QT, C::ROWS>);
    pl.lds = C::LDS + C::MORE + kKv8Deal;
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

// q4k_attn.h -- the shared-prefix attention kernel (q4k_prefix_attn.hip).
//
// A workgroup takes up to 16 * RT * WR query rows of one KV head -- for the
// prefix the rows (token, head of the group) of all requests, for a request's
// own tokens its rows -- and a stretch ("split") of the positions, and goes over
// it once with a running maximum and sum:
//   S^T = K Q^T   v_mfma_f32_16x16x32, positions x rows: a lane holds four
//                 consecutive positions of one row
//   P = exp2(c S - M)   in registers, in place: with the positions of a step
//                 of 32 numbered as two tiles of 16 hand them out, a lane's
//                 eight values are its B operand of the next product
//   O^T += V^T P^T  V read from LDS with ds_read_b64_tr_b16, which hands each
//                 lane four positions of one dimension
// so neither scores nor probabilities pass through LDS, and the running maximum
// and the sum of a row live in the lanes that hold its columns.
#pragma once

#include <hip/hip_runtime.h>

#include "q4k_batch.h"
#include "q4k_device.h"

namespace q4k {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

template <class T>
struct Vec8;
template <>
struct Vec8<_Float16> {
    typedef _Float16 type __attribute__((ext_vector_type(8)));
};
template <>
struct Vec8<__bf16> {
    typedef __bf16 type __attribute__((ext_vector_type(8)));
};

__device__ __forceinline__ f32x4 mfma(Vec8<_Float16>::type a, Vec8<_Float16>::type b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(Vec8<__bf16>::type a, Vec8<__bf16>::type b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// One cache as the kernel sees it.
struct AttnCache {
    const char *k, *v;
    int64_t k_page, k_token, k_head, v_page, v_token, v_head;  // bytes
    const int32_t *table;
    int64_t table_stride;
    int n_pages, table_len;
    int one_page;  // every position is in page `first` = table_len * r: no table, no division
    FastDiv page;
};

struct AttnParams {
    AttnCache pre, suf;
    const char *q;
    char *dst;
    float *lse;
    int64_t q_token, q_head, dst_token, dst_head;  // bytes
    const int32_t *q_start, *suffix_len;
    int n_tokens, n_requests, n_q, n_prefix, max_suffix;
    int n_head, n_head_kv, group, head_dim;
    FastDiv group_div;
    float scale;
    int q_vec;  // rows of q in 16-byte loads
    // prefix items: split, KV head, row tile (fastest); then the suffixes' items:
    // split, request, KV head, row tile
    int pre_items, pre_tiles, pre_splits, pre_len;  // pre_len, suf_len: positions of a split
    int suf_items, suf_tiles, suf_splits, suf_len;
    // partial results of `slots` splits: (M, l) and the unscaled output of every row,
    // where a second kernel joins them
    int join, slots, join_groups, join_rows;
    float2 *part_ml;
    float *part_o;
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// P is exp2(x + kBias) against the running reference, which is renewed when a
// row passes it by 2^kLazy: at most 2^15 = 32768 < F16's largest value, and F16's
// smallest step, 2^-24, is 2^-31 of the row's largest term.
constexpr float kBias = 7.0f, kLazy = 8.0f;

struct AttnSpan {
    int beg, end;         // positions
    int rows;             // query rows of the whole item's row space
    int tok0;             // first token
    int causal;           // row of token t (from tok0) sees positions < causal + t + 1 (and < end)
    int64_t table_row;    // request (prefix: 0)
    int slot;             // partial result's number
};

__device__ __forceinline__ void attn_tokens(const AttnParams &p, int r, int &t0, int &t1) {
    int64_t a = (int64_t)r * p.n_q, b = a + p.n_q;
    if (p.q_start) {
        a = p.q_start[r];
        b = p.q_start[r + 1];
        if (a < 0) a = 0;
        if (b > p.n_tokens) b = p.n_tokens;
        if (b > a + p.n_q) b = a + p.n_q;
        if (b < a) b = a;
    }
    t0 = (int)a;
    t1 = (int)b;
}
__device__ __forceinline__ int attn_suffix(const AttnParams &p, int r) {
    if (p.max_suffix == 0) return 0;
    const int n = p.suffix_len[r];
    return n < 0 ? 0 : n > p.max_suffix ? p.max_suffix : n;
}

// x as TERMS values of T whose sum is x to 11 (F16) or 8 (BF16) bits a term
template <class T, int TERMS>
__device__ __forceinline__ void split_terms(float x, T (&t)[TERMS]) {
#pragma unroll
    for (int i = 0; i < TERMS; ++i) {
        t[i] = (T)x;
        x -= (float)t[i];
    }
}

__device__ __forceinline__ float xor_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float xor_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// D: head dimension rounded up to 64, 128 or 256; RT: tiles of 16 rows per
// wave; TERMS: values of T per F32 query or probability.
template <class T, int D_, int RT_, int TERMS>
struct SharedCfg {
    using Elem = T;
    static constexpr int D = D_, RT = RT_;
    static constexpr int CH = D / 8;        // 16-byte chunks of a row of K or V
    static constexpr int RP = 256 / CH;     // rows staged per pass of the workgroup
    static constexpr int TB = 64;           // positions of a tile in LDS
    static constexpr int NP = TB / RP;      // passes
    static constexpr int ROWS = 64 * RT;
    static constexpr int LDS = 2 * TB * D * 2;
};

// Chunk swizzles.  K: 16 lanes read the same chunk of 16 rows, which go to the
// 16 bank groups of 16 bytes.  V: 32 lanes read 32 bytes of 8 rows.
template <int D>
__device__ __forceinline__ int swz_k(int t, int c) {
    return D == 64 ? c ^ ((t >> 1) & 7) : c ^ (t & 15);
}
template <int D>
__device__ __forceinline__ int swz_v(int t, int c) {
    return D == 64 ? c ^ (((t >> 1) & 3) * 2) : c ^ ((t & 7) * 2);
}

// Where a lane reads: the swizzles repeat every 16 rows, so the offsets of one
// tile of 16 positions serve all, at immediate distances.
template <int D>
struct AttnReads {
    static constexpr int NK = D / 32 < 4 ? D / 32 : 4, NV = D / 16 < 8 ? D / 16 : 8;
    int k[NK], v[NV];
    __device__ __forceinline__ AttnReads() {
        constexpr int CH = D / 8;
        const int n = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4, t = g * 4 + (n >> 2);
#pragma unroll
        for (int i = 0; i < NK; ++i) k[i] = (n * CH + swz_k<D>(n, i * 4 + g)) * 16;
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = (t * CH + swz_v<D>(t, i * 2 + ((n & 3) >> 1))) * 16 + (n & 1) * 8;
    }
    // chunk kk * 4 + g of row n of the tile at row b
    __device__ __forceinline__ int at_k(int b, int kk) const { return k[kk % NK] + kk / NK * NK * 64 + b * D * 2; }
    // dimensions dt * 16 .. of rows g * 4 .. g * 4 + 3 of the tile at row b
    __device__ __forceinline__ int at_v(int b, int dt) const { return v[dt % NV] + dt / NV * NV * 32 + b * D * 2; }
};

template <int RT, int D>
struct AttnRows {
    float c[RT];     // log2(e) * |scale| * 2^e of the row's own factor
    int limit[RT];   // positions the row sees end here
    float m[RT];     // reference in units of S; scores above `over` renew it
    float over[RT], ref[RT];  // ref: kBias - m c
    float l[RT];     // this lane's part of the sum of exp2(c s - c m + kBias)
    f32x4 o[RT][D / 16];
};

// The limits of the wave's rows row0.. and empty sums.
template <int RT, int D>
__device__ __forceinline__ void attn_rows(const AttnParams &p, const AttnSpan &s, int row0, AttnRows<RT, D> &w) {
    const int n = threadIdx.x & 15;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int row = row0 + rt * 16 + n;
        const int64_t lim = (int64_t)s.causal + (int)fastdiv((uint32_t)row, p.group_div) + 1;
        w.limit[rt] = row < s.rows && lim < s.end ? (int)lim : s.end;
        w.m[rt] = w.over[rt] = -__builtin_inff();
        w.ref[rt] = kBias;
        w.l[rt] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) w.o[rt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

// Rows row0 .. row0 + 15 of the span: dimensions kk * 32 + g * 8 .. of row n per
// lane, as TERMS values of T, handed to put(term, kk, vector).  Returns the
// row's factor c.
template <class T, int D, class QT, int TERMS, class PUT>
__device__ __forceinline__ float attn_queries(const AttnParams &p, const AttnSpan &s, int hk, int row0, PUT put) {
    using V8 = typename Vec8<T>::type;
    constexpr int KK = D / 32;
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
        const int d = kk * 32 + g * 8;
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
    if (TERMS > 1) {
        // an F32 row of any magnitude: a power of two brings its largest value to 1..2
        top = xor_max(top);
        int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
        e = e < -126 || e > 127 ? 0 : e > 126 ? 126 : e;
        f = __uint_as_float((uint32_t)(127 - e) << 23);
        c *= __uint_as_float((uint32_t)(127 + e) << 23);
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
        V8 v[TERMS];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            T t8[TERMS];
            split_terms<T, TERMS>(x[kk][j] * f, t8);
#pragma unroll
            for (int i = 0; i < TERMS; ++i) v[i][j] = t8[i];
        }
#pragma unroll
        for (int i = 0; i < TERMS; ++i) put(i, kk, v[i]);
    }
    __builtin_amdgcn_sched_barrier(0);  // one row tile's registers at a time
    // (above zero, so that c * -inf of an unseen position stays -inf at a scale of 0)
    return fmaxf(c, 1e-37f);
}

// The page of position t of the span (clamped to its last, so that nothing past a
// table is read), and the position in it.
__device__ __forceinline__ int attn_page(const AttnCache &kv, const AttnSpan &s, int t) {
    // (without a table the host has checked that a request's table_len pages are there)
    if (kv.one_page) return (int)(s.table_row * kv.table_len);
    const int e = (int)fastdiv((uint32_t)(t < s.end ? t : s.end - 1), kv.page);
    return kv.table ? kv.table[s.table_row * kv.table_stride + e] : (int)(s.table_row * kv.table_len) + e;
}
__device__ __forceinline__ int attn_slot(const AttnCache &kv, int t) {
    return kv.one_page ? t : t - (int)(fastdiv((uint32_t)t, kv.page) * kv.page.d);
}

// The first row of the item, which sees the least, sees positions below this.
template <int ROWS>
__device__ __forceinline__ int attn_least(const AttnParams &p, const AttnSpan &s, int tile) {
    const int64_t lim = (int64_t)s.causal + (int)fastdiv((uint32_t)(tile * ROWS), p.group_div) + 1;
    return lim < s.end ? (int)lim : s.end;
}

// 32 positions' scores sx[rt][tile of 16] to probabilities, in place of the next
// product's B operand.  With 16-bit queries (one term) a probability is rounded once
// to T there, the sum l takes it in F32: the result is off by 1.4 times (rms) what
// rounding it to T costs anyway (64 rows of BF16 over 32768 positions 2.3e-3 against
// 1.7e-3, F16 2.9e-4 against 2.1e-4); a second term would double the value product.
template <class T, int D, int RT, int TERMS>
__device__ __forceinline__ void attn_softmax(AttnRows<RT, D> &w, const f32x4 (&sx)[RT][2],
                                             typename Vec8<T>::type (&pf)[RT][TERMS]) {
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
    // new references when some row passes its old one by 2^kLazy (-inf: always)
    if (__any(over)) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float mn = fmaxf(w.m[rt], xor_max(top[rt]));
            // (nothing was summed yet, or nothing changes: also keeps inf - inf and 0 * inf out)
            const float f = w.m[rt] == -__builtin_inff() || w.m[rt] == mn ? 1.0f : __builtin_amdgcn_exp2f((w.m[rt] - mn) * w.c[rt]);
            w.m[rt] = mn;
            w.over[rt] = mn + kLazy / w.c[rt];
            w.ref[rt] = mn == -__builtin_inff() ? kBias : kBias - mn * w.c[rt];
            w.l[rt] *= f;
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) w.o[rt][dt] *= f;
        }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sx[rt][j >> 2][j & 3], w.c[rt], w.ref[rt]));
            w.l[rt] += x;
            T t8[TERMS];
            split_terms<T, TERMS>(x, t8);
#pragma unroll
            for (int i = 0; i < TERMS; ++i) pf[rt][i][j] = t8[i];
        }
}

// O^T += V^T P^T over 32 positions of V in LDS from row b of ldv.
template <class T, int D, int RT, int TERMS>
__device__ __forceinline__ void attn_values(AttnRows<RT, D> &w, const AttnReads<D> &rd, const typename Vec8<T>::type (&pf)[RT][TERMS],
                                            const char *ldv, int b) {
    using V8 = typename Vec8<T>::type;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) {
        union {
            s16x4 h[2];
            V8 v;
        } va;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
            va.h[tt] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4 *)(ldv + rd.at_v(b + tt * 16, dt)));
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < TERMS; ++i) w.o[rt][dt] = mfma(va.v, pf[rt][i], w.o[rt][dt]);
    }
}

// Where rows see different positions, a value of inf or NaN must not reach, as
// 0 * inf, the rows that do not see it.  There (from the first step that ends past
// `least`) such values are zeros in the products, attn_finite() says whether there
// were any, and attn_rest() adds them in the end to the rows that see them: with a
// probability above zero the sum is inf or NaN whatever the probability is.
template <class T>
__device__ __forceinline__ bool attn_finite(u32x4 &v) {
    constexpr uint32_t e = sizeof(T) == 2 && __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = (v[i] & e) == e ? 0xffffu : 0u, hi = (v[i] >> 16 & e) == e ? 0xffff0000u : 0u;
        fine = fine && (lo | hi) == 0;
        v[i] &= ~(lo | hi);
    }
    return fine;
}
template <class T, int RT, int D>
__device__ __forceinline__ void attn_rest(const AttnParams &p, const AttnCache &kv, const AttnSpan &s, int hk, AttnRows<RT, D> &w,
                                          int beg, int end) {
    const int g = (threadIdx.x & 63) >> 4;
#pragma unroll 1
    for (int t = beg; t < end; ++t) {
        const int page = attn_page(kv, s, t);
        if ((uint32_t)page >= (uint32_t)kv.n_pages) continue;
        const T *v = reinterpret_cast<const T *>(kv.v + hk * kv.v_head + page * kv.v_page + attn_slot(kv, t) * kv.v_token);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
            const int d = dt * 16 + g * 4;
            if (d >= p.head_dim) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float y = (float)v[d + j];
                if (__builtin_isfinite(y)) continue;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    if (t < w.limit[rt]) w.o[rt][dt][j] += y;
            }
        }
    }
}

// A row's reference in log2 units: its terms are exp2(log2(e) scale s - M).
__device__ __forceinline__ float attn_ref(float m, float c) { return m == -__builtin_inff() ? m : m * c - kBias; }

// Four dimensions of a row's result: to the partial results, or finished to dst
template <class QT>
__device__ __forceinline__ void attn_emit(const AttnParams &p, const AttnSpan &s, int hk, int row, int d, f32x4 x, float M, float sum) {
    if (row >= s.rows || d >= p.head_dim) return;
    const int t = (int)fastdiv((uint32_t)row, p.group_div);
    const int h = hk * p.group + row - t * p.group;
    const int64_t out = (int64_t)(s.tok0 + t) * p.n_head + h;
    if (p.join) {
        const int64_t at = (int64_t)s.slot * p.n_tokens * p.n_head + out;
        if (d == 0) p.part_ml[at] = make_float2(M, sum);
        *reinterpret_cast<f32x4 *>(p.part_o + at * p.head_dim + d) = x;
        return;
    }
    if (d == 0 && p.lse) p.lse[out] = sum == 0.0f ? -__builtin_inff() : (M + log2f(sum)) * kLn2;
    QT *dst = reinterpret_cast<QT *>(p.dst + (int64_t)(s.tok0 + t) * p.dst_token + h * p.dst_head) + d;
#pragma unroll
    for (int j = 0; j < 4; ++j) dst[j] = (QT)(sum == 0.0f ? 0.0f : x[j] / sum);
}

// ---- few rows: every wave takes all of them over positions of its own ----
// A wave's 32 rows of K, then of V, pass through LDS that belongs to it: whole
// rows come from memory in 16-byte pieces that neighbouring lanes read side by
// side (read in the operand's layout they would be 64 separate pieces a load), and
// waves never wait for each other before the end.  Memory bound: each wave keeps
// the next 32 positions' K and V on their way.  24 rows over 131072 positions of 8
// heads of 128 BF16 dimensions (537 MB): 113 us, 4.8 TB/s with F32 queries as three
// terms.  64 F16 rows over 8192 positions and 16 x 256 of their own, with the join:
// 22.2 us, of which about 5 read memory: bound by the four steps' round trips.  Of 256
// dimensions they spill 20 bytes a lane, one workgroup a CU as it is.
template <class T, int D_, int RT_, int TERMS>
struct StreamCfg {
    using Elem = T;
    static constexpr int D = D_, RT = RT_, ROWS = 16 * RT_;
    // Queries of 32 registers and more stay in LDS: held in registers they spill
    // beside two steps' K and V (64 F16 rows over 65536 positions: 76 / 65 us).
    static constexpr bool QLDS = D_ / 32 * RT_ * TERMS >= 8;
    static constexpr int VBYTES = 4 * 32 * D * 2;  // (and a row tile's outputs of four waves at the end)
    static constexpr int QBYTES = QLDS ? RT * TERMS * (D / 32) * 1024 : 0;  // (else they pass through V's place)
    static constexpr int LDS = VBYTES * 2 > 64 * D * 4 ? VBYTES + QBYTES : 64 * D * 4 + QBYTES;
};

template <class C, class QT, int TERMS>
__device__ __forceinline__ void attn_stream(const AttnParams &p, const AttnCache &kv, const AttnSpan &s, int hk, int tile,
                                            char *lds, int *flags) {
    using T = typename C::Elem;
    using V8 = typename Vec8<T>::type;
    constexpr int D = C::D, RT = C::RT, KK = D / 32, CH = D / 8;
    constexpr int RI = 64 / CH, NI = 32 / RI;  // rows of a load, loads of 32 rows
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int row0 = tile * C::ROWS;
    char *ldw = lds + wave * 32 * D * 2;
    char *ldq = lds + (C::QLDS ? C::LDS - C::QBYTES : 0);
    AttnRows<RT, D> w;
    V8 q[C::QLDS ? 1 : RT][TERMS][KK];
    const int least = attn_least<C::ROWS>(p, s, tile);

    // lane: chunk lane % CH of rows i * RI + lane / CH
    const int sc = lane % CH, sr = lane / CH;
    const bool cok = sc * 8 < p.head_dim;  // (past the head: chunk 0 again, as zeros in K; V's are not stored)
    const char *kb = kv.k + hk * kv.k_head + (cok ? sc * 16 : 0), *vb = kv.v + hk * kv.v_head + (cok ? sc * 16 : 0);
    // where each of the 32 rows begins, in K and V: lane r works out row r, all read it
    longlong2 *rows = reinterpret_cast<longlong2 *>(reinterpret_cast<char *>(flags) + 1024) + wave * 32;
    u32x4 kf[NI], vf[NI];
    uint32_t there = 0;  // bit r: position r of the step that was loaded has a page
    int page;
    auto load_k = [&](int t0) {
        const int t = t0 + (lane & 31);
        const bool ok = t < s.end && (uint32_t)page < (uint32_t)kv.n_pages;
        there = (uint32_t)__ballot(ok);
        const int pg = ok ? page : 0, slot = ok ? attn_slot(kv, t) : 0;
        if (lane < 32) rows[lane] = make_longlong2(pg * kv.k_page + slot * kv.k_token, pg * kv.v_page + slot * kv.v_token);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < NI; ++i) kf[i] = *reinterpret_cast<const u32x4 *>(kb + rows[i * RI + sr].x);
    };
    auto load_v = [&]() {
#pragma unroll
        for (int i = 0; i < NI; ++i) vf[i] = *reinterpret_cast<const u32x4 *>(vb + rows[i * RI + sr].y);
    };
    int t0 = s.beg + wave * 32;
    if (t0 < s.end) {
        page = attn_page(kv, s, t0 + (lane & 31));
        load_k(t0);
        load_v();
        page = attn_page(kv, s, t0 + 128 + (lane & 31));
    }
    // the queries, one row tile per wave, while the first positions are on their way
    attn_rows<RT, D>(p, s, row0, w);
    float *cs = reinterpret_cast<float *>(flags);
    if (wave < RT) {
        const float c = attn_queries<T, D, QT, TERMS>(p, s, hk, row0 + wave * 16, [&](int i, int kk, V8 v) {
            *reinterpret_cast<V8 *>(ldq + ((wave * TERMS + i) * KK + kk) * 1024 + lane * 16) = v;
        });
        if (g == 0) cs[wave * 16 + n] = c;
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) w.c[rt] = cs[rt * 16 + n];
    if (!C::QLDS) {
#pragma unroll
        for (int f = 0; f < RT * TERMS * KK; ++f)
            q[C::QLDS ? 0 : f / (TERMS * KK)][f / KK % TERMS][f % KK] = *reinterpret_cast<const V8 *>(ldq + f * 1024 + lane * 16);
        __syncthreads();
    }
    const AttnReads<D> rd;
    const u32x4 zero = {0, 0, 0, 0};
    bool fine = true;  // of the values at and after the first step that ends past `least`
    for (; t0 < s.end; t0 += 128) {
        const uint32_t ok = there;
        const bool careful = least < s.end && t0 + 32 > least;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = i * RI + sr;
            *reinterpret_cast<u32x4 *>(ldw + (r * CH + swz_k<D>(r, sc)) * 16) = cok ? kf[i] : zero;
        }
        // The next step's K leaves before this one's scores (own positions only: 43.5 us
        // after them, 42.6 so).  No branch, or the waits for these loads would be for
        // all of them: past the end no position is there.
        load_k(t0 + 128);
        page = attn_page(kv, s, t0 + 256 + (lane & 31));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // rows are written before lanes read each other's
        f32x4 sx[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sx[rt][0] = sx[rt][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            V8 ka[2];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) ka[tt] = *reinterpret_cast<const V8 *>(ldw + rd.at_k(tt * 16, kk));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int i = 0; i < TERMS; ++i) {
                    const V8 qv = C::QLDS ? *reinterpret_cast<const V8 *>(ldq + ((rt * TERMS + i) * KK + kk) * 1024 + lane * 16)
                                          : q[C::QLDS ? 0 : rt][i][kk];
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt) sx[rt][tt] = mfma(ka[tt], qv, sx[rt][tt]);
                }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (careful) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const bool here = (ok >> (i * RI + sr)) & 1;
                fine = (attn_finite<T>(vf[i]) || !here) && fine;
            }
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r = i * RI + sr;
            // (a position that is not there: values of zero, whatever was read)
            *reinterpret_cast<u32x4 *>(ldw + (r * CH + swz_v<D>(r, sc)) * 16) = (ok >> r) & 1 ? vf[i] : zero;
        }
        load_v();
        if (careful || ok != 0xffffffffu) {
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int u = tt * 16 + g * 4 + j;
                        if (!((ok >> u) & 1) || t0 + u >= w.limit[rt]) sx[rt][tt][j] = -__builtin_inff();
                    }
        }
        V8 pf[RT][TERMS];
        attn_softmax<T, D, RT, TERMS>(w, sx, pf);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        attn_values<T, D, RT, TERMS>(w, rd, pf, ldw, 0);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if (!__all(fine))
        for (t0 = s.beg + wave * 32; t0 < s.end; t0 += 128)
            if (t0 + 32 > least) attn_rest<T>(p, kv, s, hk, w, t0, t0 + 32 < s.end ? t0 + 32 : s.end);

    // the four waves' parts of each row tile join in LDS
    float *ol = reinterpret_cast<float *>(lds);        // [wave][16][D]
    float2 *ml = reinterpret_cast<float2 *>(flags);    // [wave][16]
    constexpr int Q4 = D / 4;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = xor_sum(w.l[rt]);
        __syncthreads();
        if (g == 0) ml[wave * 16 + n] = make_float2(attn_ref(w.m[rt], w.c[rt]), sum);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt)
            *reinterpret_cast<f32x4 *>(ol + (wave * 16 + n) * D + (((dt * 4 + g) ^ n) * 4)) = w.o[rt][dt];
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
            attn_emit<QT>(p, s, hk, row0 + rt * 16 + r, d4 * 4, acc, M, ls);
        }
    }
}

// ---- many rows: the waves take rows of their own and share K and V in LDS ----
// 512 rows over 32768 positions of 8 heads of 128 BF16 dimensions: 69 GFLOP in 108 us
// with the join (635 TFLOP/s), over 131072 in 337 us (816; a large library product
// reaches 1217).  The
// softmax's vector work (exponentials a quarter rate) takes 30 % of the time, the
// matrix cores 20 %, LDS 20 %; two workgroups a CU, whose registers allow no third,
// do not overlap them fully.  Tiles of 64 rows per wave do not fit the registers, nor
// do F32 queries on F16 at 128 dimensions: their two terms a query take the 256
// registers and 36 to 48 bytes of scratch a lane.
template <class C, class QT, int TERMS>
__device__ __forceinline__ void attn_shared(const AttnParams &p, const AttnCache &kv, const AttnSpan &s, int hk, int tile,
                                            char *lds, int *flags) {
    using T = typename C::Elem;
    using V8 = typename Vec8<T>::type;
    constexpr int D = C::D, RT = C::RT, CH = C::CH, RP = C::RP, TB = C::TB, NP = C::NP;
    constexpr int KK = D / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const char *ldk = lds;
    const char *ldv = lds + TB * D * 2;
    uint8_t *seen = reinterpret_cast<uint8_t *>(flags + 4);  // one byte per position of the tile
    AttnRows<RT, D> w;
    V8 q[RT][TERMS][KK];
    const int row0 = tile * C::ROWS + wave * RT * 16;
    attn_rows<RT, D>(p, s, row0, w);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
        w.c[rt] = attn_queries<T, D, QT, TERMS>(p, s, hk, row0 + rt * 16, [&](int i, int kk, V8 v) { q[rt][i][kk] = v; });
    const int least = attn_least<C::ROWS>(p, s, tile);

    // staging: thread -> chunk tid % CH of positions tid / CH + RP * i
    const int sc = tid % CH, sr = tid / CH;
    const bool cok = sc * 8 < p.head_dim;
    const char *kb = kv.k + hk * kv.k_head + (cok ? sc * 16 : 0), *vb = kv.v + hk * kv.v_head + (cok ? sc * 16 : 0);
    const int64_t first = kv.one_page ? s.table_row * kv.table_len : 0, one = first * kv.k_page, one_v = first * kv.v_page;
    u32x4 kr[NP], vr[NP];
    int page[NP];        // of the tile that is loaded next
    uint32_t okbits = 0; // which of this thread's positions have a page
    auto get_pages = [&](int t0) {
#pragma unroll
        for (int i = 0; i < NP; ++i) page[i] = attn_page(kv, s, t0 + sr + RP * i);
    };
    auto load = [&](int t0) {
        if (kv.one_page && t0 + TB <= s.end) {
            // one stretch of memory: a row's place is the first one's and a constant
            const char *k0 = kb + one + (int64_t)(t0 + sr) * kv.k_token, *v0 = vb + one_v + (int64_t)(t0 + sr) * kv.v_token;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                kr[i] = *reinterpret_cast<const u32x4 *>(k0 + i * (RP * kv.k_token));
                vr[i] = *reinterpret_cast<const u32x4 *>(v0 + i * (RP * kv.v_token));
            }
            okbits = (1u << NP) - 1;
            return;
        }
        okbits = 0;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int t = t0 + sr + RP * i;
            const bool ok = t < s.end && (uint32_t)page[i] < (uint32_t)kv.n_pages;
            const int pg = ok ? page[i] : 0, slot = ok ? attn_slot(kv, t) : 0;
            kr[i] = *reinterpret_cast<const u32x4 *>(kb + pg * kv.k_page + slot * kv.k_token);
            vr[i] = *reinterpret_cast<const u32x4 *>(vb + pg * kv.v_page + slot * kv.v_token);
            okbits |= (uint32_t)ok << i;
        }
    };
    if (s.beg < s.end) {
        get_pages(s.beg);
        load(s.beg);
        get_pages(s.beg + TB);
    }
    if (tid == 0) flags[0] = flags[2] = 0;

    const AttnReads<D> rd;
    int par = 0;
    for (int t0 = s.beg; t0 < s.end; t0 += TB, par ^= 1) {
        __syncthreads();  // the last tile is no longer read
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int t = sr + RP * i;
            const bool ok = (okbits >> i) & 1;
            if (least < s.end && t0 + TB > least && ok && !attn_finite<T>(vr[i])) flags[2] = 1;  // (stays for the end)
            const u32x4 zero = {0, 0, 0, 0};
            // (past the head: zeros for the queries' zeros; a position that is not there: values of zero)
            *reinterpret_cast<u32x4 *>(lds + (t * CH + swz_k<D>(t, sc)) * 16) = cok ? kr[i] : zero;
            *reinterpret_cast<u32x4 *>(lds + TB * D * 2 + (t * CH + swz_v<D>(t, sc)) * 16) = ok ? vr[i] : zero;
            if (sc == 0) seen[t] = ok;
        }
        // flags[par]: some position of this tile is not seen.  The other word, read
        // before the barrier above, is cleared for the next tile.
        if (okbits != (1u << NP) - 1) flags[par] = 1;
        if (tid == 0) flags[par ^ 1] = 0;
        const int tn = t0 + TB;
        if (tn < s.end) {
            load(tn);
            get_pages(tn + TB);
        }
        __syncthreads();
        const bool masked = flags[par] != 0 || t0 + TB > least;

#pragma unroll
        for (int b = 0; b < TB; b += 32) {
            f32x4 sx[RT][2];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) sx[rt][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    const V8 ka = *reinterpret_cast<const V8 *>(ldk + rd.at_k(b + tt * 16, kk));
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int i = 0; i < TERMS; ++i) sx[rt][tt] = mfma(ka, q[rt][i][kk], sx[rt][tt]);
                }
            }
            if (masked) {
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const int t = b + tt * 16 + g * 4;
                    const uint32_t ok4 = *reinterpret_cast<const uint32_t *>(seen + t);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (!((ok4 >> (8 * j)) & 1) || t0 + t + j >= w.limit[rt]) sx[rt][tt][j] = -__builtin_inff();
                }
            }
            V8 pf[RT][TERMS];
            attn_softmax<T, D, RT, TERMS>(w, sx, pf);
            // (ahead of the other workgroup's softmax, which fills the gaps: 148 -> 142 us for
            // 64 requests of 64 heads behind 32768 tokens)
            __builtin_amdgcn_s_setprio(1);
            attn_values<T, D, RT, TERMS>(w, rd, pf, ldv, b);
            __builtin_amdgcn_s_setprio(0);
        }
    }
    __syncthreads();
    if (flags[2] != 0) {
        int t = s.beg;
        while (t + TB <= least) t += TB;
        attn_rest<T>(p, kv, s, hk, w, t, s.end);
    }
    // through LDS, so that rows are stored by lanes side by side
    float *ol = reinterpret_cast<float *>(lds);        // [wave][16][D]
    float2 *ml = reinterpret_cast<float2 *>(flags);    // [wave][16]
    constexpr int Q4 = D / 4;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = xor_sum(w.l[rt]);
        __syncthreads();
        if (g == 0) ml[wave * 16 + n] = make_float2(attn_ref(w.m[rt], w.c[rt]), sum);
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt)
            *reinterpret_cast<f32x4 *>(ol + (wave * 16 + n) * D + (((dt * 4 + g) ^ n) * 4)) = w.o[rt][dt];
        __syncthreads();
#pragma unroll 2
        for (int x = tid; x < 64 * Q4; x += 256) {
            const int r = x / Q4, d4 = x % Q4;
            const float2 e = ml[r];
            attn_emit<QT>(p, s, hk, tile * C::ROWS + (r / 16 * RT + rt) * 16 + r % 16, d4 * 4,
                          *reinterpret_cast<const f32x4 *>(ol + r * D + ((d4 ^ (r & 15)) * 4)), e.x, e.y);
        }
    }
}

template <class T, int D, int RT, int TERMS, class QT>
__device__ __forceinline__ void attn_item(StreamCfg<T, D, RT, TERMS>, const AttnParams &p, const AttnCache &kv, const AttnSpan &s,
                                          int hk, int tile, char *lds, int *flags, QT) {
    attn_stream<StreamCfg<T, D, RT, TERMS>, QT, TERMS>(p, kv, s, hk, tile, lds, flags);
}
template <class T, int D, int RT, int TERMS, class QT>
__device__ __forceinline__ void attn_item(SharedCfg<T, D, RT, TERMS>, const AttnParams &p, const AttnCache &kv, const AttnSpan &s,
                                          int hk, int tile, char *lds, int *flags, QT) {
    attn_shared<SharedCfg<T, D, RT, TERMS>, QT, TERMS>(p, kv, s, hk, tile, lds, flags);
}

// Consecutive items to one XCD (workgroups go to the 8 XCDs in turn), so that the
// row tiles of one stretch of the cache read it through one L2.
__device__ __forceinline__ int xcd_item(int b, int total) {
    const int per = total / 8, more = total % 8, x = b % 8;
    return x * per + (x < more ? x : more) + b / 8;
}

// bytes after the tiles: flags, or (M, l) of four waves' rows; where the rows of four waves begin
constexpr int kAttnFlags = 1024 + 2048;

// CP: how the prefix's rows are taken, CS the suffixes'.
template <class CP, class CS, class QT, int TERMS>
__global__ __launch_bounds__(256, CP::D == 256 ? 1 : 2) void prefix_attn_kernel(AttnParams p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int buf = CP::LDS > CS::LDS ? CP::LDS : CS::LDS;
    int *flags = reinterpret_cast<int *>(lds + buf);
    AttnSpan s;
    if ((int)blockIdx.x < p.pre_items) {
        const int item = xcd_item(blockIdx.x, p.pre_items);
        const int tile = item % p.pre_tiles, x = item / p.pre_tiles;
        const int hk = x % p.n_head_kv, sp = x / p.n_head_kv;
        s.beg = sp * p.pre_len;
        s.end = s.beg + p.pre_len < p.n_prefix ? s.beg + p.pre_len : p.n_prefix;
        s.rows = p.n_tokens * p.group;
        s.tok0 = 0;
        s.causal = p.n_prefix;
        s.table_row = 0;
        s.slot = sp;
        attn_item(CP(), p, p.pre, s, hk, tile, lds, flags, QT());
        return;
    }
    const int item = xcd_item(blockIdx.x - p.pre_items, p.suf_items);
    const int tile = item % p.suf_tiles;
    int x = item / p.suf_tiles;
    const int hk = x % p.n_head_kv;
    x /= p.n_head_kv;
    const int r = x % p.n_requests, sp = x / p.n_requests;
    int t0, t1;
    attn_tokens(p, r, t0, t1);
    const int len = attn_suffix(p, r);
    s.beg = sp * p.suf_len;
    // (the first split of a request that sees nothing writes its empty rows when nothing else would)
    if (s.beg >= len && (p.join || sp > 0)) return;
    s.end = s.beg + p.suf_len < len ? s.beg + p.suf_len : len;
    s.rows = (t1 - t0) * p.group;
    s.tok0 = t0;
    s.causal = len - (t1 - t0);
    s.table_row = r;
    s.slot = p.pre_splits + sp;
    if (tile * CS::ROWS >= s.rows) return;
    attn_item(CS(), p, p.suf, s, hk, tile, lds, flags, QT());
}

// Joins the partial results of p.join_rows rows per workgroup of 256: groups of
// head_dim / 4 lanes, p.join_groups of them to a row, take every join_groups-th
// split with a running reference, so that nothing waits for a first pass over the
// references.
template <class QT>
__global__ __launch_bounds__(256) void prefix_attn_join_kernel(AttnParams p) {
    __shared__ f32x4 acc[256];
    __shared__ float2 mls[256];
    const int q4 = p.head_dim / 4;
    const int grp = threadIdx.x / q4, d4 = threadIdx.x - grp * q4;
    const int sub = grp % p.join_groups, which = grp / p.join_groups;
    const int item = blockIdx.x * p.join_rows + which;
    const int rt = item / p.n_head, head = item - rt * p.n_head;
    const int r = rt / p.n_q, t = rt - r * p.n_q;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f, M = -__builtin_inff();
    // A split in which the row sees nothing (l of 0) adds nothing, whatever its values.
    auto add = [&](float2 e, f32x4 x) {
        if (e.y == 0.0f) return;
        const float mn = fmaxf(M, e.x);
        const float f = M == mn || l == 0.0f ? 1.0f : __builtin_amdgcn_exp2f(M - mn);
        const float g = e.x == mn ? 1.0f : __builtin_amdgcn_exp2f(e.x - mn);
        l = l * f + e.y * g;
        o = o * f + x * g;
        M = mn;
    };
    int tok = -1;
    if (which < p.join_rows && r < p.n_requests) {
        int t0, t1;
        attn_tokens(p, r, t0, t1);
        if (t0 + t < t1) tok = t0 + t;
    }
    const int64_t row = (int64_t)tok * p.n_head + head, step = (int64_t)p.n_tokens * p.n_head;
    if (tok >= 0) {
        const int len = attn_suffix(p, r);
        const int n = p.pre_splits + (p.suf_len > 0 ? (len + p.suf_len - 1) / p.suf_len : 0);
        constexpr int U = 4;
        for (int i0 = sub; i0 < n; i0 += p.join_groups * U) {
            float2 e[U];
            f32x4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t at = (i0 + u * p.join_groups < n ? i0 + u * p.join_groups : i0) * step + row;
                e[u] = p.part_ml[at];
                x[u] = *reinterpret_cast<const f32x4 *>(p.part_o + at * p.head_dim + d4 * 4);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i0 + u * p.join_groups < n) add(e[u], x[u]);
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
    if (d4 == 0 && p.lse) p.lse[row] = l == 0.0f ? -__builtin_inff() : (M + log2f(l)) * kLn2;
}

// ---- which kernel runs a call ----
struct AttnPlan {
    int dim, pre_size, suf_size;  // padded head dimension, shapes
    AttnParams p;
    size_t bytes;
    int lds;
    const void *kernel;
};

// (an instantiation of attn_kernel_of per pair of types, each in a file of its own)
void attn_kernel_f16(AttnPlan &pl);
void attn_kernel_f16_f32(AttnPlan &pl);
void attn_kernel_bf16(AttnPlan &pl);
void attn_kernel_bf16_f32(AttnPlan &pl);

// How rows are taken: 0 and 1 streaming 16 and 32 rows, 2 sharing K and V
// among four waves of RT tiles of 16 rows.
template <class T, int D, int TERMS, int SIZE>
struct AttnShape {
    using cfg = StreamCfg<T, D, SIZE == 1 && D < 256 ? 2 : 1, TERMS>;
};
template <class T, int D, int TERMS>
struct AttnShape<T, D, TERMS, 2> {
    using cfg = SharedCfg<T, D, D < 256 ? 2 : 1, TERMS>;
};


template <class T, class QT, int TERMS, int D, int PS, int SS>
void attn_kernel(AttnPlan &pl) {
    using CP = typename AttnShape<T, D, TERMS, PS>::cfg;
    using CS = typename AttnShape<T, D, TERMS, SS>::cfg;
    pl.kernel = reinterpret_cast<const void *>(&prefix_attn_kernel<CP, CS, QT, TERMS>);
    pl.lds = (CP::LDS > CS::LDS ? CP::LDS : CS::LDS) + kAttnFlags;
}
template <class T, class QT, int TERMS, int D>
void attn_kernel_of(AttnPlan &pl) {
    // (three terms a query and up to 128 dimensions: streaming only)
    constexpr int most = TERMS == 3 && D < 256 ? 1 : 2;
    switch (pl.pre_size * 4 + pl.suf_size) {
        case 0: return attn_kernel<T, QT, TERMS, D, 0, 0>(pl);
        case 4: return attn_kernel<T, QT, TERMS, D, 1, 0>(pl);
        case 5: return attn_kernel<T, QT, TERMS, D, 1, 1>(pl);
        case 8: return attn_kernel<T, QT, TERMS, D, most, 0>(pl);
        case 9: return attn_kernel<T, QT, TERMS, D, most, 1>(pl);
        default: return attn_kernel<T, QT, TERMS, D, most, most>(pl);
    }
}
template <class T, class QT, int TERMS>
void attn_kernel_of(AttnPlan &pl) {
    if (pl.dim == 64) attn_kernel_of<T, QT, TERMS, 64>(pl);
    else if (pl.dim == 128) attn_kernel_of<T, QT, TERMS, 128>(pl);
    else attn_kernel_of<T, QT, TERMS, 256>(pl);
}

}  // namespace q4k

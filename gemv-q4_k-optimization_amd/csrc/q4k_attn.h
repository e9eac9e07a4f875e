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

#include "q4k_batch_host.h"
#include "q4k_device.h"

namespace q4k {

typedef float f32x4 __attribute__((ext_vector_type(4)));
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
    // prefix items: split, KV head, row tile (fastest); then the suffixes' items:
    // split, request, KV head, row tile
    int pre_items, pre_tiles, pre_splits, pre_len;  // pre_len, suf_len: positions of a split
    int suf_items, suf_tiles, suf_splits, suf_len;
    // partial results of `slots` splits: (M, l) and the unscaled output of every row
    int slots;
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
// wave; WR: waves over rows, the others of the four over positions; TERMS:
// values of T per F32 query or probability.
template <class T, int D_, int RT_, int WR_>
struct AttnCfg {
    using Elem = T;
    static constexpr int D = D_, RT = RT_, WR = WR_, WT = 4 / WR_;
    static constexpr int CH = D / 8;        // 16-byte chunks of a row of K or V
    static constexpr int RP = 256 / CH;     // rows staged per pass of the workgroup
    static constexpr int TB = D == 256 ? 64 : WT == 1 ? 64 : 128;  // positions of a tile in LDS
    static constexpr int NP = TB / RP;      // passes
    static constexpr int ROWS = 16 * RT * WR;
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

template <class C, class QT, int TERMS>
__device__ __forceinline__ void attn_span(const AttnParams &p, const AttnCache &kv, const AttnSpan &s, int hk, int tile0,
                                          char *lds, int *flags) {
    using T = typename C::Elem;
    using V8 = typename Vec8<T>::type;
    constexpr int D = C::D, RT = C::RT, WT = C::WT, CH = C::CH, RP = C::RP, TB = C::TB, NP = C::NP;
    constexpr int KK = D / 32, DT = D / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int wr = wave / WT, wt = wave % WT;
    const char *ldk = lds;
    const char *ldv = lds + TB * D * 2;
    uint8_t *seen = reinterpret_cast<uint8_t *>(flags + 4);  // one byte per position of the tile

    // ---- queries: lane n of a tile's rows, eight dimensions each ----
    V8 q[RT][TERMS][KK];
    float c[RT];       // log2(e) * scale, and 2^e of the row's own factor
    int limit[RT];     // positions the row sees end here
    const float sgn = p.scale < 0.0f ? -1.0f : 1.0f;
    const int row0 = tile0 * C::ROWS + wr * RT * 16;
    int lim_min = s.end;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int row = row0 + rt * 16 + n;
        const bool ok = row < s.rows;
        const int t = (int)fastdiv((uint32_t)(ok ? row : 0), p.group_div);
        const int h = hk * p.group + (ok ? row : 0) - t * p.group;
        const QT *src = reinterpret_cast<const QT *>(p.q + (int64_t)(s.tok0 + t) * p.q_token + h * p.q_head);
        const int64_t lim = (int64_t)s.causal + t + 1;
        limit[rt] = lim < s.end ? (int)lim : s.end;
        if (!ok) limit[rt] = s.end;
        float x[KK][8];
        float top = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int d = kk * 32 + g * 8 + j;
                x[kk][j] = ok && d < p.head_dim ? (float)src[d] * sgn : 0.0f;
                top = fmaxf(top, fabsf(x[kk][j]));
            }
        c[rt] = fabsf(p.scale) * kLog2e;
        float f = 1.0f;
        if (TERMS > 1) {
            // an F32 row of any magnitude: a power of two brings its largest value to 1..2
            top = xor_max(top);
            int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
            e = e < -126 || e > 127 ? 0 : e > 126 ? 126 : e;
            f = __uint_as_float((uint32_t)(127 - e) << 23);
            c[rt] *= __uint_as_float((uint32_t)(127 + e) << 23);
        }
        // (above zero, so that c * -inf of an unseen position stays -inf at a scale of 0)
        c[rt] = fmaxf(c[rt], 1e-37f);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                T t8[TERMS];
                split_terms<T, TERMS>(x[kk][j] * f, t8);
#pragma unroll
                for (int i = 0; i < TERMS; ++i) q[rt][i][kk][j] = t8[i];
            }
    }
    {
        // the first row of the workgroup sees the least
        const int t = (int)fastdiv((uint32_t)(tile0 * C::ROWS), p.group_div);
        const int64_t lim = (int64_t)s.causal + t + 1;
        if (lim < lim_min) lim_min = (int)lim;
    }

    f32x4 o[RT][DT];
    float m[RT], l[RT];  // m: reference in units of S; l: this lane's part of the sum
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -__builtin_inff();
        l[rt] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[rt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // ---- staging: thread -> chunk tid % CH of positions tid / CH + RP * i ----
    const int sc = tid % CH, sr = tid / CH;
    const bool cok = sc * 8 < p.head_dim;
    const char *kb = kv.k + hk * kv.k_head + sc * 16, *vb = kv.v + hk * kv.v_head + sc * 16;
    u32x4 kr[NP], vr[NP];
    int page[NP];   // of the tile that is loaded next; -1: not seen
    auto get_pages = [&](int t0) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int t = t0 + sr + RP * i;
            page[i] = -1;
            if (t < s.end) {
                if (kv.one_page) {
                    page[i] = (int)s.table_row * kv.table_len;
                } else {
                    const int e = (int)fastdiv((uint32_t)t, kv.page);
                    page[i] = kv.table ? kv.table[s.table_row * kv.table_stride + e] : (int)s.table_row * kv.table_len + e;
                }
            }
        }
    };
    auto load = [&](int t0) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            kr[i] = u32x4{0, 0, 0, 0};
            vr[i] = u32x4{0, 0, 0, 0};
            const int t = t0 + sr + RP * i;
            if ((uint32_t)page[i] < (uint32_t)kv.n_pages && cok) {
                const int slot = kv.one_page ? t : t - (int)(fastdiv((uint32_t)t, kv.page) * kv.page.d);
                kr[i] = *reinterpret_cast<const u32x4 *>(kb + page[i] * kv.k_page + slot * kv.k_token);
                vr[i] = *reinterpret_cast<const u32x4 *>(vb + page[i] * kv.v_page + slot * kv.v_token);
            }
        }
    };
    uint32_t okbits = 0;  // which of this thread's positions have a page
    auto get_okbits = [&]() {
        okbits = 0;
#pragma unroll
        for (int i = 0; i < NP; ++i) okbits |= (uint32_t)((uint32_t)page[i] < (uint32_t)kv.n_pages) << i;
    };
    get_pages(s.beg);
    load(s.beg);
    get_okbits();
    get_pages(s.beg + TB);
    if (tid == 0) flags[0] = 0;

    int par = 0;
    for (int t0 = s.beg; t0 < s.end; t0 += TB, par ^= 1) {
        __syncthreads();  // the last tile is no longer read
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int t = sr + RP * i;
            *reinterpret_cast<u32x4 *>(lds + (t * CH + swz_k<D>(t, sc)) * 16) = kr[i];
            *reinterpret_cast<u32x4 *>(lds + TB * D * 2 + (t * CH + swz_v<D>(t, sc)) * 16) = vr[i];
            if (sc == 0) seen[t] = (okbits >> i) & 1;
        }
        // flags[par]: some position of this tile is not seen.  The other word, read
        // before the barrier above, is cleared for the next tile.
        if (okbits != (1u << NP) - 1) flags[par] = 1;
        if (tid == 0) flags[par ^ 1] = 0;
        const int tn = t0 + TB;
        if (tn < s.end) {
            load(tn);
            get_okbits();
            get_pages(tn + TB);
        }
        __syncthreads();
        const bool masked = flags[par] != 0 || t0 + TB > lim_min;

#pragma unroll 1
        for (int st = wt; st < TB / 32; st += WT) {
            const int b = st * 32;
            if (t0 + b >= s.end) break;
            f32x4 sx[RT][2];
#pragma unroll
            for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) sx[rt][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                const int t = b + tt * 16 + n;
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    const V8 ka = *reinterpret_cast<const V8 *>(ldk + (t * CH + swz_k<D>(t, kk * 4 + g)) * 16);
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
                            if (!((ok4 >> (8 * j)) & 1) || t0 + t + j >= limit[rt]) sx[rt][tt][j] = -__builtin_inff();
                }
            }
            V8 pf[RT][TERMS];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                float top = sx[rt][0][0];
#pragma unroll
                for (int j = 1; j < 8; ++j) top = fmaxf(top, sx[rt][j >> 2][j & 3]);
                // a new reference when some row passes the old one by 2^kLazy (-inf: always)
                if (__any((top - m[rt]) * c[rt] > kLazy || m[rt] == -__builtin_inff())) {
                    const float mn = fmaxf(m[rt], xor_max(top));
                    // (nothing was summed yet, or nothing changes: also keeps inf - inf and 0 * inf out)
                    const float f = m[rt] == -__builtin_inff() || m[rt] == mn ? 1.0f : __builtin_amdgcn_exp2f((m[rt] - mn) * c[rt]);
                    m[rt] = mn;
                    l[rt] *= f;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) o[rt][dt] *= f;
                }
                const float ref = m[rt] == -__builtin_inff() ? kBias : kBias - m[rt] * c[rt];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sx[rt][j >> 2][j & 3], c[rt], ref));
                    l[rt] += x;
                    T t8[TERMS];
                    split_terms<T, TERMS>(x, t8);
#pragma unroll
                    for (int i = 0; i < TERMS; ++i) pf[rt][i][j] = t8[i];
                }
            }
            const int tr = b + g * 4 + (n >> 2);
            auto load_v = [&](int dt) {
                union {
                    s16x4 h[2];
                    V8 v;
                } va;
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const int t = tr + tt * 16;
                    va.h[tt] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s16x4 *)(ldv + (t * CH + swz_v<D>(t, dt * 2 + ((n & 3) >> 1))) * 16 +
                                                                    (n & 1) * 8));
                }
                return va.v;
            };
            // Where rows see different positions, a value of inf or NaN must not
            // reach (as 0 * inf) the rows that do not see it.
            bool odd = false;
            if (t0 + b + 32 > lim_min) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    const V8 va = load_v(dt);
#pragma unroll
                    for (int j = 0; j < 8; ++j) odd |= !__builtin_isfinite((float)va[j]);
                }
            }
            if (__any(odd)) {
                // the finite values for all rows, then the others one position at a
                // time, kept only by the rows that see it
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    V8 va = load_v(dt);
#pragma unroll
                    for (int j = 0; j < 8; ++j) va[j] = __builtin_isfinite((float)va[j]) ? va[j] : (T)0.0f;
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int i = 0; i < TERMS; ++i) o[rt][dt] = mfma(va, pf[rt][i], o[rt][dt]);
                }
#pragma unroll 1
                for (int u = 0; u < 32; ++u) {
                    const bool mine = g == ((u & 15) >> 2);
                    const int ju = (u >> 4) * 4 + (u & 3);
                    const bool there = seen[b + u] != 0;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        V8 va = load_v(dt);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            va[j] = mine && j == ju && !__builtin_isfinite((float)va[j]) ? va[j] : (T)0.0f;
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            f32x4 x = o[rt][dt];
#pragma unroll
                            for (int i = 0; i < TERMS; ++i) {
                                V8 pu = pf[rt][i];
#pragma unroll
                                for (int j = 0; j < 8; ++j) pu[j] = mine && j == ju ? pu[j] : (T)0.0f;
                                x = mfma(va, pu, x);
                            }
                            if (there && t0 + b + u < limit[rt]) o[rt][dt] = x;
                        }
                    }
                }
                continue;
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const V8 va = load_v(dt);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int i = 0; i < TERMS; ++i) o[rt][dt] = mfma(va, pf[rt][i], o[rt][dt]);
            }
        }
    }

    // ---- the row's sum over its four lane groups; waves over positions join in LDS ----
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] = xor_sum(l[rt]);
    // M in log2 units: the row's terms are exp2(log2(e) scale s - M)
    auto emit = [&](int row, int d, f32x4 x, float M, float sum) {
        if (row >= s.rows || d >= p.head_dim) return;
        const int t = (int)fastdiv((uint32_t)row, p.group_div);
        const int h = hk * p.group + row - t * p.group;
        const int64_t out = (int64_t)(s.tok0 + t) * p.n_head + h;
        if (p.slots > 1) {
            const int64_t at = (int64_t)s.slot * p.n_tokens * p.n_head + out;
            if (d == 0) p.part_ml[at] = make_float2(M, sum);
            *reinterpret_cast<f32x4 *>(p.part_o + at * p.head_dim + d) = x;
            return;
        }
        if (d == 0 && p.lse) p.lse[out] = sum == 0.0f ? -__builtin_inff() : (M + log2f(sum)) * kLn2;
        QT *dst = reinterpret_cast<QT *>(p.dst + (int64_t)(s.tok0 + t) * p.dst_token + h * p.dst_head) + d;
#pragma unroll
        for (int j = 0; j < 4; ++j) dst[j] = (QT)(sum == 0.0f ? 0.0f : x[j] / sum);
    };
    if (WT == 1) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const float M = m[rt] == -__builtin_inff() ? m[rt] : m[rt] * c[rt] - kBias;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) emit(row0 + rt * 16 + n, dt * 16 + g * 4, o[rt][dt], M, l[rt]);
        }
        return;
    }
    __syncthreads();
    float *ol = reinterpret_cast<float *>(lds);                 // [wave][RT * 16][D]
    float2 *ml = reinterpret_cast<float2 *>(flags + 4);         // [wave][RT * 16]
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = wave * RT * 16 + rt * 16 + n;
        if (g == 0) ml[r] = make_float2(m[rt] == -__builtin_inff() ? m[rt] : m[rt] * c[rt] - kBias, l[rt]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
            *reinterpret_cast<f32x4 *>(ol + r * D + (((dt * 4 + g) ^ n) * 4)) = o[rt][dt];
    }
    __syncthreads();
    constexpr int Q4 = D / 4;
    for (int x = tid; x < C::ROWS * Q4; x += 256) {
        const int r = x / Q4, d4 = x % Q4;
        const int w0 = r / (RT * 16) * WT, rr = r % (RT * 16);
        float M = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < WT; ++w) M = fmaxf(M, ml[(w0 + w) * RT * 16 + rr].x);
        f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
        float ls = 0.0f;
#pragma unroll
        for (int w = 0; w < WT; ++w) {
            const float2 e = ml[(w0 + w) * RT * 16 + rr];
            if (e.y == 0.0f) continue;  // no position of the row in this wave's part
            const float f = __builtin_amdgcn_exp2f(e.x == M ? 0.0f : e.x - M);
            ls += e.y * f;
            sum += *reinterpret_cast<const f32x4 *>(ol + ((w0 + w) * RT * 16 + rr) * D + ((d4 ^ (rr & 15)) * 4)) * f;
        }
        emit(tile0 * C::ROWS + r, d4 * 4, sum, M, ls);
    }
}

// Consecutive items to one XCD (workgroups go to the 8 XCDs in turn), so that the
// row tiles of one stretch of the cache read it through one L2.
__device__ __forceinline__ int xcd_item(int b, int total) {
    const int per = total / 8, more = total % 8, x = b % 8;
    return x * per + (x < more ? x : more) + b / 8;
}

// CP: rows and waves of the prefix's items, CS of the suffixes'.
template <class CP, class CS, class QT, int TERMS>
__global__ __launch_bounds__(256) void prefix_attn_kernel(AttnParams p) {
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
        attn_span<CP, QT, TERMS>(p, p.pre, s, hk, tile, lds, flags);
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
    if (s.beg >= len && (p.slots > 1 || sp > 0)) return;
    s.end = s.beg + p.suf_len < len ? s.beg + p.suf_len : len;
    s.rows = (t1 - t0) * p.group;
    s.tok0 = t0;
    s.causal = len - (t1 - t0);
    s.table_row = r;
    s.slot = p.pre_splits + sp;
    if (tile * CS::ROWS >= s.rows) return;
    attn_span<CS, QT, TERMS>(p, p.suf, s, hk, tile, lds, flags);
}

// Joins a row's partial results: one workgroup of 256 per row, groups of
// head_dim / 4 lanes taking every 256 / (head_dim / 4)-th split.
template <class QT>
__global__ __launch_bounds__(256) void prefix_attn_join_kernel(AttnParams p) {
    __shared__ f32x4 acc[256];
    const int head = blockIdx.x % p.n_head;
    const int rt = blockIdx.x / p.n_head;
    const int r = rt / p.n_q, t = rt - r * p.n_q;
    int t0, t1;
    attn_tokens(p, r, t0, t1);
    const int tok = t0 + t;
    if (tok >= t1) return;
    const int len = attn_suffix(p, r);
    const int n = p.pre_splits + (p.suf_len > 0 ? (len + p.suf_len - 1) / p.suf_len : 0);
    const int64_t row = (int64_t)tok * p.n_head + head, step = (int64_t)p.n_tokens * p.n_head;
    const int lane = threadIdx.x & 63;
    float M = -__builtin_inff();
    for (int i = lane; i < n; i += 64) M = fmaxf(M, p.part_ml[i * step + row].x);
#pragma unroll
    for (int x = 1; x < 64; x *= 2) M = fmaxf(M, __shfl_xor(M, x));
    const int q4 = p.head_dim / 4, per = 256 / q4;
    const int grp = threadIdx.x / q4, d4 = threadIdx.x % q4;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
    if (grp < per) {
#pragma unroll 4
        for (int i = grp; i < n; i += per) {
            const float2 e = p.part_ml[i * step + row];
            const f32x4 x = *reinterpret_cast<const f32x4 *>(p.part_o + (i * step + row) * p.head_dim + d4 * 4);
            // (a split in which the row sees nothing adds nothing, whatever its values)
            const float f = __builtin_amdgcn_exp2f(e.x == M ? 0.0f : e.x - M);
            if (e.y != 0.0f) {
                l += e.y * f;
                o += x * f;
            }
        }
    }
    __shared__ float ls[256];
    acc[threadIdx.x] = o;
    ls[threadIdx.x] = l;
    __syncthreads();
    if (threadIdx.x >= q4) return;
    for (int i = 1; i < per; ++i) {
        o += acc[i * q4 + d4];
        l += ls[i * q4 + d4];
    }
    QT *dst = reinterpret_cast<QT *>(p.dst + tok * p.dst_token + head * p.dst_head) + d4 * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) dst[j] = (QT)(l == 0.0f ? 0.0f : o[j] / l);
    if (threadIdx.x == 0 && p.lse) p.lse[row] = l == 0.0f ? -__builtin_inff() : (M + log2f(l)) * kLn2;
}

}  // namespace q4k

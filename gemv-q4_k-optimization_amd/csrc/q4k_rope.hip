// q4k_rope.hip -- q4k_rope (include/q4k_step.h): RMS norms of queries and keys for
// each head and the rotation by their positions, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * w            (where the rows have a norm)
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t)   for the pairs of a head
//
// A wave takes heads of one token.  A lane holds both values of its pairs -- four
// of the first and four of the second member where rows allow it -- so nothing
// moves between lanes but the sum of squares, and works out the cosines of its
// token once for all its heads: lane i those of pair i, from pos * freq in turns in
// 64 bits, less the whole quarter turns before it is rounded.
//
// Many tokens are bound by memory: 4096 tokens of 64 + 8 heads of 128 with norms, F32 to BF16,
// 226 MB, take 49 us, 4.6 TB/s (a large copy: 5.2).  One token takes 3.6 us, a launch's own time.
// Rows that do not allow four values at once pay for it twice over: 4096 tokens of 64 + 8 heads of 80, 142 MB,
// 103 us with 20 of the dimensions rotated, 38 with 32.
#include <hip/hip_runtime.h>

#include <cmath>

#include "../../include/q4k_step.h"
#include "q4k_batch.h"
#include "q4k_device.h"

namespace q4k {

struct RopePart {
    const char *src;
    char *dst;
    const float *norm;
    int64_t src_token, src_head, dst_token, dst_head;
};
struct RopeParams {
    RopePart q, k;
    const int32_t *pos;
    const float *factors;
    int n_q, n_head;  // heads of the queries, of both
    int n_tokens, chunks, per;  // heads' rounds of a wave, waves of a token
    int head_dim, n_rot;
    bool past;  // results go past the caches
    float eps, magnitude;
    double turns[Q4K_ROPE_MAX_HEAD_DIM / 2];  // of a pair per position
};

template <int W, class T>
struct RopeVec {
    typedef T type __attribute__((ext_vector_type(W)));
    typedef __attribute__((address_space(1))) type global;
};
template <class T>
struct RopeVec<1, T> {
    typedef T type;
    typedef __attribute__((address_space(1))) T global;
};
template <int W, class T>
__device__ __forceinline__ void rope_store(char *p, const float *x, bool past) {
    union {
        T e[W];
        typename RopeVec<W, T>::type v;
    } u;
#pragma unroll
    for (int j = 0; j < W; ++j) u.e[j] = (T)x[j];
    auto *to = (typename RopeVec<W, T>::global *)p;
    if (past) {
        __builtin_nontemporal_store(u.v, to);
    } else {
        asm volatile("");  // (on both sides, or the compiler makes the two stores one, of this kind)
        *to = u.v;
        asm volatile("");
    }
}

// cos and sin of a whole turn times `turns`
__device__ __forceinline__ float2 rope_angle(double turns) {
    double a = turns - rint(turns);   // -1/2 .. 1/2
    const double quarter = rint(a * 4.0);
    const float r = (float)(a * 4.0 - quarter);  // of a quarter turn, -1/2 .. 1/2
    float s, c;
    sincospif(0.5f * r, &s, &c);
    switch ((int)quarter & 3) {
        case 0: return make_float2(c, s);
        case 1: return make_float2(-s, c);
        case 2: return make_float2(-c, -s);
        default: return make_float2(s, -c);
    }
}

// The values in scalar registers: a choice between two parts' else becomes each lane's own load
// of what it chose, round by round.  (What comes out are addresses of no known memory: loads and stores
// say that theirs is global.  4096 x 72 heads: 59.8 us, 51.2 so).
__device__ __forceinline__ RopePart rope_scalars(RopePart r) {
    asm("" : "+s"(r.src), "+s"(r.dst), "+s"(r.src_token), "+s"(r.src_head), "+s"(r.dst_token), "+s"(r.dst_head));
    return r;
}

// W: pairs of a unit (a lane's two pieces of W values), NU: units of a lane; LANES:
// lanes of a head, a power of two.
template <int W, int NU, int LANES, bool NEOX, class S, class D>
__global__ __launch_bounds__(256) void rope_kernel(RopeParams p) {
    constexpr int HEADS = 64 / LANES;  // of a wave's round
    __shared__ float2 table[4][Q4K_ROPE_MAX_HEAD_DIM / 2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int item = blockIdx.x * 4 + wave;
    const int tok = item / p.chunks, chunk = item - tok * p.chunks;
    const bool there = tok < p.n_tokens;
    const RopePart q = rope_scalars(p.q), k = rope_scalars(p.k);
    const int sub = lane % LANES;
    const int half = p.n_rot / 2;

    // the unit's pieces: places of values, and the first of its pairs (half and
    // above: not rotated)
    int at[NU][2], pair[NU];
    bool in[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const int i = (sub + u * LANES) * W;  // pairs before this unit
        in[u] = 2 * i < p.head_dim;
        pair[u] = i;
        if (NEOX && i < half) {
            at[u][0] = i;
            at[u][1] = half + i;
        } else {
            at[u][0] = 2 * i;
            at[u][1] = 2 * i + W;
        }
    }
    // (as they are in memory: a conversion would wait for them; where there is nothing: the row's first
    // values, or the first row's)
    union Pieces {
        typename RopeVec<W, S>::type v[2];
        S e[2 * W];
    } pieces[NU];
    auto load = [&](int round) {
        const int head = round * HEADS + lane / LANES;
        const bool ok = there && head < p.n_head, isq = head < p.n_q || (!ok && p.n_q > 0);
        const char *row = isq ? q.src : k.src;
        if (ok) row += isq ? tok * q.src_token + head * q.src_head : tok * k.src_token + (head - p.n_q) * k.src_head;
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                pieces[u].v[i] = *(const typename RopeVec<W, S>::global *)(row + (in[u] ? at[u][i] : 0) * sizeof(S));
    };
    int round = chunk * p.per;
    const int rounds = (p.n_head + HEADS - 1) / HEADS, end = round + p.per < rounds ? round + p.per : rounds;
    load(round);
    const int pos = there ? p.pos[tok] : 0;
    for (int i = lane; i < half; i += 64) {
        double t = (double)pos * p.turns[i];
        if (p.factors) t /= (double)p.factors[i];
        table[wave][i] = rope_angle(t);
    }
    float w[2][NU][2 * W];
    const bool norms = p.q.norm || p.k.norm;
    if (norms) {
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int j = 0; j < 2 * W; ++j) {
                const int d = in[u] ? at[u][j / W] + j % W : 0;
                w[0][u][j] = p.q.norm ? p.q.norm[d] : 1.0f;
                w[1][u][j] = p.k.norm ? p.k.norm[d] : 1.0f;
            }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's own table is written
    float2 cs[NU][W];
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int j = 0; j < W; ++j) {
            cs[u][j] = pair[u] + j < half ? table[wave][pair[u] + j] : make_float2(1.0f, 0.0f);
            if (pair[u] + j < half) {
                cs[u][j].x *= p.magnitude;
                cs[u][j].y *= p.magnitude;
            }
        }
    // (a second round on its way beside the one in hand: 52.6 us)
    for (;;) {
        float x[NU][2 * W];
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int j = 0; j < 2 * W; ++j) x[u][j] = in[u] ? (float)pieces[u].e[j] : 0.0f;
        const int head = round * HEADS + lane / LANES;
        const bool isq = head < p.n_q;
        if (norms) {
            float sum = 0.0f;
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int j = 0; j < 2 * W; ++j) sum = __builtin_fmaf(x[u][j], x[u][j], sum);
#pragma unroll
            for (int o = LANES / 2; o > 0; o /= 2) sum += __shfl_xor(sum, o);
            // (rows without a norm: times 1)
            const bool have = isq ? p.q.norm != nullptr : p.k.norm != nullptr;
            const float r = have ? 1.0f / sqrtf(sum / (float)p.head_dim + p.eps) : 1.0f;
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int j = 0; j < 2 * W; ++j) x[u][j] = x[u][j] * r * (isq ? w[0][u][j] : w[1][u][j]);
        }
        if (there && head < p.n_head) {
            char *row = isq ? q.dst + tok * q.dst_token + head * q.dst_head : k.dst + tok * k.dst_token + (head - p.n_q) * k.dst_head;
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                if (!in[u]) continue;
                float y[2 * W];
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    // pair j: (j, W + j) of halves, (2j, 2j + 1) of neighbours; where
                    // nothing turns either way is the same
                    const int i0 = NEOX ? j : 2 * j, i1 = NEOX ? W + j : 2 * j + 1;
                    const float a = x[u][i0], b = x[u][i1];
                    const float2 t = cs[u][j];
                    y[i0] = a * t.x - b * t.y;
                    y[i1] = a * t.y + b * t.x;
                }
                if (pair[u] >= half)
#pragma unroll
                    for (int j = 0; j < 2 * W; ++j) y[j] = x[u][j];
                rope_store<W, D>(row + at[u][0] * sizeof(D), y, p.past);
                rope_store<W, D>(row + at[u][1] * sizeof(D), y + W, p.past);
            }
        }
        if (++round >= end) break;
        load(round);
    }
}

static int rope_size(int32_t type) { return type == Q4K_GGML_TYPE_F32 ? 4 : 2; }

static bool rope_rows_ok(const q4k_rope_rows &r, int64_t n_tokens, int head_dim) {
    const bool f32 = r.src_type == Q4K_GGML_TYPE_F32;
    if (!f32 && r.src_type != Q4K_GGML_TYPE_F16 && r.src_type != Q4K_GGML_TYPE_BF16) return false;
    if (r.dst_type != r.src_type && !(f32 && (r.dst_type == Q4K_GGML_TYPE_F16 || r.dst_type == Q4K_GGML_TYPE_BF16))) return false;
    const int ss = rope_size(r.src_type), ds = rope_size(r.dst_type);
    if (r.n_head < 0 || !aligned(r.norm, 4)) return false;
    if (r.n_head == 0 || n_tokens == 0) return true;
    if (!r.src || !r.dst || !aligned(r.src, ss) || !aligned(r.dst, ds)) return false;
    if (((r.nb_src_token | r.nb_src_head) & (ss - 1)) || ((r.nb_dst_token | r.nb_dst_head) & (ds - 1))) return false;
    if (r.n_head > 1 && (r.nb_src_head < (int64_t)ss * head_dim || r.nb_dst_head < (int64_t)ds * head_dim)) return false;
    if (n_tokens > 1 && (r.nb_dst_token < (int64_t)ds * head_dim)) return false;
    // in place: the same type and strides
    if (r.src == r.dst && (ss != ds || r.nb_src_token != r.nb_dst_token || r.nb_src_head != r.nb_dst_head)) return false;
    return true;
}
static bool rope_rows_vec(const q4k_rope_rows &r) {
    const int s = 4 * rope_size(r.src_type), d = 4 * rope_size(r.dst_type);
    return aligned(r.src, s) && aligned(r.dst, d) && ((r.nb_src_token | r.nb_src_head) & (s - 1)) == 0 &&
           ((r.nb_dst_token | r.nb_dst_head) & (d - 1)) == 0;
}

using RopeFn = void (*)(RopeParams);
template <bool NEOX, class S, class D>
static RopeFn rope_fn(int dim, bool vec, int &lanes) {
    if (vec) {
        const int units = (dim + 7) / 8;
        lanes = units <= 8 ? 8 : units <= 16 ? 16 : 32;
        return lanes == 8 ? rope_kernel<4, 1, 8, NEOX, S, D> : lanes == 16 ? rope_kernel<4, 1, 16, NEOX, S, D> : rope_kernel<4, 1, 32, NEOX, S, D>;
    }
    lanes = 64;
    return dim <= 128 ? rope_kernel<1, 1, 64, NEOX, S, D> : rope_kernel<1, 2, 64, NEOX, S, D>;
}
template <bool NEOX>
static RopeFn rope_fn(int src_type, int dst_type, int dim, bool vec, int &lanes) {
    if (src_type == Q4K_GGML_TYPE_F32)
        return dst_type == Q4K_GGML_TYPE_F32   ? rope_fn<NEOX, float, float>(dim, vec, lanes)
               : dst_type == Q4K_GGML_TYPE_F16 ? rope_fn<NEOX, float, _Float16>(dim, vec, lanes)
                                               : rope_fn<NEOX, float, __bf16>(dim, vec, lanes);
    return src_type == Q4K_GGML_TYPE_F16 ? rope_fn<NEOX, _Float16, _Float16>(dim, vec, lanes) : rope_fn<NEOX, __bf16, __bf16>(dim, vec, lanes);
}

// One launch over the queries' and the keys' rows where their types agree.
static int rope_launch(RopeParams &p, const q4k_rope_rows *q, const q4k_rope_rows *k, bool neox, int cus, void *stream) {
    auto part = [](const q4k_rope_rows *r) {
        return r ? RopePart{(const char *)r->src, (char *)r->dst, r->norm, r->nb_src_token, r->nb_src_head, r->nb_dst_token, r->nb_dst_head}
                 : RopePart{};
    };
    p.q = part(q);
    p.k = part(k);
    p.n_q = q ? (int)q->n_head : 0;
    p.n_head = p.n_q + (k ? (int)k->n_head : 0);
    // Pieces of four values where every row allows them, else single values.
    const bool vec = (!q || rope_rows_vec(*q)) && (!k || rope_rows_vec(*k)) && p.n_rot % 8 == 0 && p.head_dim % 8 == 0;
    const q4k_rope_rows &any = q ? *q : *k;
    int lanes;
    const RopeFn fn = neox ? rope_fn<true>(any.src_type, any.dst_type, p.head_dim, vec, lanes) : rope_fn<false>(any.src_type, any.dst_type, p.head_dim, vec, lanes);
    // (kStreamFloats: 4096 x 72 heads of 128 to BF16, 75 MB, 52.8 us into the caches, 46.0 past them)
    p.past = p.n_tokens * (int64_t)p.n_head * p.head_dim * rope_size(any.dst_type) >= kStreamFloats * 4;
    // A round of a wave's heads each where tokens are few; the more rounds of a token
    // the fewer times its cosines are worked out, while 16 waves a CU remain.
    const int heads = 64 / lanes;
    const int64_t rounds = (p.n_head + heads - 1) / heads;
    int64_t per = p.n_tokens * rounds / (16 * (int64_t)cus);
    per = per < 1 ? 1 : per > rounds ? rounds : per;
    p.per = (int)per;
    p.chunks = (int)((rounds + per - 1) / per);
    if (p.n_tokens > ((int64_t)INT32_MAX - 4) / p.chunks) return Q4K_EUNSUPPORTED;
    return launch(fn, dim3((unsigned)(((int64_t)p.n_tokens * p.chunks + 3) / 4)), 256, 0, stream, p);
}

}  // namespace q4k

using namespace q4k;

extern "C" int q4k_rope(const q4k_rope_args *args, void *stream) {
    if (!args) return Q4K_EINVAL;
    const q4k_rope_args &a = *args;
    if (a.head_dim < 1 || a.n_rot < 0 || a.n_rot > a.head_dim || a.n_rot % 2 != 0 || a.n_tokens < 0 || a.n_tokens > INT32_MAX) return Q4K_EINVAL;
    if (a.mode != Q4K_ROPE_NORMAL && a.mode != Q4K_ROPE_NEOX) return Q4K_EINVAL;
    if (!(a.freq_base > 0.0f) || !std::isfinite(a.freq_base) || !std::isfinite(a.freq_scale) || !std::isfinite(a.ext_factor) ||
        !std::isfinite(a.attn_factor) || !(a.eps >= 0.0f))
        return Q4K_EINVAL;
    if (a.ext_factor != 0.0f && (!(a.freq_base > 1.0f) || !(a.freq_scale > 0.0f) || !(a.beta_fast > 0.0f) || !(a.beta_slow > 0.0f) || a.n_ctx_orig < 1))
        return Q4K_EINVAL;
    if (!aligned(a.freq_factors, 4) || !aligned(a.pos, 4)) return Q4K_EINVAL;
    const q4k_rope_rows *q = a.q, *k = a.k;
    if ((q && !rope_rows_ok(*q, a.n_tokens, a.head_dim)) || (k && !rope_rows_ok(*k, a.n_tokens, a.head_dim))) return Q4K_EINVAL;
    if (q && q->n_head == 0) q = nullptr;
    if (k && k->n_head == 0) k = nullptr;
    if (a.n_tokens == 0 || (!q && !k)) return Q4K_OK;
    if (!a.pos) return Q4K_EINVAL;
    if (a.head_dim % 2 != 0 || a.head_dim > Q4K_ROPE_MAX_HEAD_DIM) return Q4K_EUNSUPPORTED;
    // (heads of both are counted in 31 bits, up to a round past the last one)
    if ((q ? q->n_head : 0) > (1 << 29) || (k ? k->n_head : 0) > (1 << 29)) return Q4K_EUNSUPPORTED;
    DeviceInfo *di;
    int st = device_info(&di);
    if (st != Q4K_OK) return st;
    RopeParams p{};
    p.pos = a.pos;
    p.factors = a.freq_factors;
    p.n_tokens = (int)a.n_tokens;
    p.head_dim = a.head_dim;
    p.n_rot = a.n_rot;
    const bool neox = a.mode == Q4K_ROPE_NEOX;
    p.eps = a.eps;
    double m = a.attn_factor, lo = 0.0, hi = 0.0;
    constexpr double two_pi = 6.283185307179586476925;
    if (a.ext_factor != 0.0f) {
        m *= 1.0 - 0.1 * std::log((double)a.freq_scale);
        // the pair that turns `beta` times over the original context
        auto pair_of = [&](double beta) { return 0.5 * a.n_rot * std::log(a.n_ctx_orig / (beta * two_pi)) / std::log((double)a.freq_base); };
        lo = std::fmax(0.0, std::floor(pair_of(a.beta_fast)));
        hi = std::fmin(a.n_rot - 1.0, std::ceil(pair_of(a.beta_slow)));
    }
    p.magnitude = (float)m;
    // (a running product, off by up to a half step of 64 bits a factor; pos * turns is rounded once more: some 1e-6
    // of a radian at position 2^31, 1e-9 at 2^20, where F32's rounding of an angle below 1 is 6e-8)
    double f = 1.0 / two_pi;
    const double step = a.n_rot > 0 ? std::exp2(-2.0 / a.n_rot * std::log2((double)a.freq_base)) : 1.0;
    for (int i = 0; i < a.n_rot / 2; ++i, f *= step) {
        double s = a.freq_scale;
        if (a.ext_factor != 0.0f) {
            const double y = (i - lo) / std::fmax(0.001, hi - lo);
            const double r = a.ext_factor * (1.0 - std::fmin(1.0, std::fmax(0.0, y)));
            s = s * (1.0 - r) + r;
        }
        p.turns[i] = f * s;
    }
    if (q && k && (q->src_type != k->src_type || q->dst_type != k->dst_type)) {
        st = rope_launch(p, q, nullptr, neox, di->cus, stream);
        return st == Q4K_OK ? rope_launch(p, nullptr, k, neox, di->cus, stream) : st;
    }
    return rope_launch(p, q, k, neox, di->cus, stream);
}

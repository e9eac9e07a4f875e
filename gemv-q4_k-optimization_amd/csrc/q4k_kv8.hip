// q4k_kv8.hip -- q4k_kv8_store and q4k_kv8_load (include/q4k_step.h): keys and
// values into pages of 8 bits with a scale for each block of tokens and head, and
// back.
//
//   store   s' = max(s if the block holds earlier tokens, max |x| / top), 1 where that is 0 and some |x| infinite
//           q = rne(x / s') for new tokens; earlier ones rne(q s / s') where s' > s
//   load    x = q s
//
// A workgroup stores the new tokens of one block and head, keys or values: one pass
// over its rows for the magnitude, held in registers for the rounding.
//
// Bound by chains of round trips (lengths, page, rows and scale, stores): one token of 16 requests 4.4 us
// to store, 4.4 to load, a launch's own time; 8 x 512 BF16 tokens of 8 heads of 128 to e4m3, 25 MB, 13.1 to 13.5 us,
// 5.6 of which are the rounding's vector work, and back, 25 MB, 7.4 to 7.8 us.
#include "q4k_kv8.h"

namespace q4k {

struct Kv8RowsParams {
    Kv8Cache c;
    Kv8Tokens t;
    char *k, *v;  // rows
    int64_t k_token, k_head, v_token, v_head;
    int n_head, head_dim, blocks;  // blocks: that a request's new tokens may lie in
};

// x / s to the nearest value of 8 bits, ties to even, of a scale s >= 0.  A quotient
// that F32 cannot hold goes to the neighbour whose last bit is 1 (the remainder, which
// fma gives exactly, tells the side), so that it can neither become a tie nor
// leave one when it is rounded again.  Either neighbour will do to begin with, so that
// of scales whose remainders are no subnormals 1 / s and one step of Newton's take the
// division's place (8 x 512 tokens of 8 heads of 128: the whole store 13.5 us, 15.8 with divisions and loads one by one).
template <bool I8>
struct Kv8Scale {
    static constexpr float top = I8 ? 127.0f : 448.0f;
    float s, inverse, most;
    bool usual;
    __device__ __forceinline__ explicit Kv8Scale(float x) : s(x), inverse(1.0f / x), most(2.0f * top * x), usual(x > 0x1p-80f && x < 0x1p100f) {}
    __device__ __forceinline__ static float odd(float y, float rest) {
        const uint32_t bits = __float_as_uint(y);
        return rest != 0.0f && y != 0.0f && (bits & 1) == 0 ? __uint_as_float((rest > 0.0f) == (y > 0.0f) ? bits + 1 : bits - 1) : y;
    }
    __device__ __forceinline__ float round(float x) const {
        float y = 0.0f;
        if (usual) {
            x = x == x ? fminf(fmaxf(x, -most), most) : 0.0f;
            y = x * inverse;
            y = __builtin_fmaf(__builtin_fmaf(-y, s, x), inverse, y);
            y = odd(y, __builtin_fmaf(-y, s, x));
        } else if (__builtin_isinf(x)) {
            y = x;
        } else if (x == x && s > 0.0f) {
            y = x / s;
            y = odd(y, __builtin_fmaf(-y, s, x));
        }
        y = fminf(fmaxf(y, -top), top);
        return I8 ? rintf(y) : y;
    }
};
template <bool I8>
__device__ __forceinline__ uint32_t kv8_pack(const float (&y)[4]) {
    if (I8) return ((int)y[0] & 255) | ((int)y[1] & 255) << 8 | ((int)y[2] & 255) << 16 | (uint32_t)(int)y[3] << 24;
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}
template <bool I8>
__device__ __forceinline__ void kv8_unpack(uint32_t w, float (&x)[4]) {
    if (I8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = (float)(int8_t)(w >> (8 * j));
    } else {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        x[0] = a[0];
        x[1] = a[1];
        x[2] = b[0];
        x[3] = b[1];
    }
}
// four values of T at any address of T's alignment
template <class T>
__device__ __forceinline__ void kv8_row4(const char *p, float (&x)[4]) {
    typedef T vec __attribute__((ext_vector_type(4)));
    typedef vec any __attribute__((aligned(sizeof(T))));
    const vec v = *reinterpret_cast<const any *>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (float)v[j];
}

template <int THREADS, bool I8, class T>
__global__ __launch_bounds__(THREADS) void kv8_store_kernel(Kv8RowsParams p) {
    constexpr int HELD = 8;  // rows of a thread in registers
    const int tid = threadIdx.x;
    // items: block of the request, head, keys or values (fastest)
    const bool isv = blockIdx.x & 1;
    int x = blockIdx.x >> 1;
    const int h = x % p.n_head;
    x /= p.n_head;
    const int r = x / p.blocks, j = x - r * p.blocks;
    int t0, t1, len;
    kv8_tokens(p.t, r, t0, t1, len);
    const int first = len - (t1 - t0), from = first < 0 ? 0 : first;
    const int block = (int)p.c.block.d;
    const int64_t b0 = ((int64_t)fastdiv((uint32_t)from, p.c.block) + j) * block;  // the block's first position
    if (b0 >= len || t1 == t0) return;
    const int beg = from > b0 ? from : (int)b0, end = b0 + block < len ? (int)b0 + block : len;
    const int page = kv8_page(p.c, r, (int)b0);
    if (beg >= end || (uint32_t)page >= (uint32_t)p.c.n_pages) return;
    const int slot = (int)b0 - (int)(fastdiv((uint32_t)b0, p.c.page) * p.c.page.d);  // of the page
    char *held = (isv ? p.c.v + page * p.c.v_page + h * p.c.v_head : p.c.k + page * p.c.k_page + h * p.c.k_head);
    const int64_t held_token = isv ? p.c.v_token : p.c.k_token;
    float *scale_at = reinterpret_cast<float *>(reinterpret_cast<char *>(isv ? p.c.v_scale : p.c.k_scale) + page * p.c.s_page +
                                                (int64_t)fastdiv((uint32_t)slot, p.c.block) * p.c.s_block + h * p.c.s_head);
    const char *rows = (isv ? p.v + h * p.v_head : p.k + h * p.k_head);
    const int64_t row_token = isv ? p.v_token : p.k_token;

    const int d4 = p.head_dim / 4, per = THREADS / d4;  // lanes of a row, rows of a pass
    const int sub = tid / d4, d = (tid - sub * d4) * 4;
    const bool on = sub < per;
    const int64_t tok = (int64_t)t0 + (beg - first);  // the row of position beg
    const float was = b0 < beg ? *scale_at : 0.0f;
    float xs[HELD][4];
    float top = 0.0f;
    auto row_of = [&](int i) { return rows + (tok + i) * row_token + d * sizeof(T); };
    // (past the last row that one again, without branches, in which each load would be waited for by itself)
#pragma unroll
    for (int i = 0; i < HELD; ++i) kv8_row4<T>(row_of(i * per + sub < end - beg ? i * per + sub : end - beg - 1), xs[i]);
#pragma unroll
    for (int i = 0; i < HELD; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (__builtin_isfinite(xs[i][e])) top = fmaxf(top, fabsf(xs[i][e]));
    for (int at = HELD * per + sub; on && at < end - beg; at += per) {
        float y[4];
        kv8_row4<T>(row_of(at), y);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (__builtin_isfinite(y[e])) top = fmaxf(top, fabsf(y[e]));
    }
#pragma unroll
    for (int o = 32; o > 0; o /= 2) top = fmaxf(top, __shfl_xor(top, o));
    if (THREADS > 64) {
        __shared__ float tops[THREADS / 64];
        if ((tid & 63) == 0) tops[tid >> 6] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < THREADS / 64; ++i) top = fmaxf(top, tops[i]);
    }
    float s = fmaxf(top / Kv8Scale<I8>::top, was);
    if (s == 0.0f) {
        // Nothing to take a scale from: 1 where there is an infinity, so that it reads back as the largest
        // of its sign.
        bool inf = false;
#pragma unroll
        for (int i = 0; i < HELD; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) inf |= __builtin_isinf(xs[i][e]);
        for (int at = HELD * per + sub; on && at < end - beg; at += per) {
            float y[4];
            kv8_row4<T>(row_of(at), y);
#pragma unroll
            for (int e = 0; e < 4; ++e) inf |= __builtin_isinf(y[e]);
        }
        if (__syncthreads_or(inf)) s = 1.0f;
    }
    const Kv8Scale<I8> by(s);
    const bool grows = !(s <= was);
    auto put = [&](int position, const float (&y)[4]) {
        float q[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = by.round(y[e]);
        *reinterpret_cast<uint32_t *>(held + (slot + (position - (int)b0)) * held_token + d) = kv8_pack<I8>(q);
    };
    if (b0 < beg && grows)
        for (int at = sub; on && at < beg - (int)b0; at += per) {
            float y[4];
            kv8_unpack<I8>(*reinterpret_cast<const uint32_t *>(held + (slot + at) * held_token + d), y);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] *= was;
            put((int)b0 + at, y);
        }
    if (tid == 0 && (b0 == beg || grows)) *scale_at = s;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int at = i * per + sub;
        if (on && at < end - beg) put(beg + at, xs[i]);
    }
    for (int at = HELD * per + sub; on && at < end - beg; at += per) {
        float y[4];
        kv8_row4<T>(row_of(at), y);
        put(beg + at, y);
    }
}

// Eight values of a row and head per thread, of keys and values.
template <bool I8, class T>
__global__ __launch_bounds__(256) void kv8_load_kernel(Kv8RowsParams p) {
    const int d8 = p.head_dim / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)p.t.n_requests * p.t.n_q;
    const int64_t rh = i / d8;
    const int d = (int)(i - rh * d8) * 8;
    const int64_t row = rh / p.n_head;
    const int h = (int)(rh - row * p.n_head);
    if (row >= rows) return;
    const int r = (int)(row / p.t.n_q), t = (int)(row - (int64_t)r * p.t.n_q);
    int t0, t1, len;
    kv8_tokens(p.t, r, t0, t1, len);
    if (t >= t1 - t0) return;
    const int position = len - (t1 - t0) + t;
    const int page = position < 0 ? -1 : kv8_page(p.c, r, position);
    const bool there = (uint32_t)page < (uint32_t)p.c.n_pages;
    const int slot = there ? position - (int)(fastdiv((uint32_t)position, p.c.page) * p.c.page.d) : 0;
    const int64_t s_at = there ? page * p.c.s_page + (int64_t)fastdiv((uint32_t)slot, p.c.block) * p.c.s_block + h * p.c.s_head : 0;
    auto one = [&](char *dst, const char *held, const float *scale) {
        uint2 w = make_uint2(0, 0);
        float s = 0.0f;
        if (there) {
            w = *reinterpret_cast<const uint2 *>(held + d);
            s = *reinterpret_cast<const float *>(reinterpret_cast<const char *>(scale) + s_at);
        }
        float x[2][4];
        kv8_unpack<I8>(w.x, x[0]);
        kv8_unpack<I8>(w.y, x[1]);
        typedef T vec __attribute__((ext_vector_type(4)));
        typedef vec any __attribute__((aligned(sizeof(T))));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            vec y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = there ? (T)(x[u][e] * s) : (T)0.0f;
            reinterpret_cast<any *>(dst + d * sizeof(T))[u] = y;
        }
    };
    const int64_t tok = t0 + t;
    if (p.k)
        one(p.k + tok * p.k_token + h * p.k_head, p.c.k + (there ? page * p.c.k_page + slot * p.c.k_token + h * p.c.k_head : 0), p.c.k_scale);
    if (p.v)
        one(p.v + tok * p.v_token + h * p.v_head, p.c.v + (there ? page * p.c.v_page + slot * p.c.v_token + h * p.c.v_head : 0), p.c.v_scale);
}

static bool kv8_row_ok(const void *p, int64_t token, int64_t head, int es, const q4k_kv8_pages &c) {
    if (!p) return true;
    return aligned(p, es) && ((token | head) & (es - 1)) == 0 && (c.n_head_kv == 1 || head >= (int64_t)es * c.head_dim);
}

// Rows of `bytes` that one step of a stride apart do not overlap, where there is more than one: what
// workgroups write at once.
static bool kv8_apart(int64_t stride, int64_t n, int64_t bytes) { return n <= 1 || stride >= bytes || stride <= -bytes; }
static bool kv8_writable(const q4k_kv8_pages &c) {
    const int64_t blocks = c.page_size / c.block;
    return kv8_apart(c.nb_k_page, c.n_pages, c.head_dim) && kv8_apart(c.nb_k_token, c.page_size, c.head_dim) && kv8_apart(c.nb_k_head, c.n_head_kv, c.head_dim) &&
           kv8_apart(c.nb_v_page, c.n_pages, c.head_dim) && kv8_apart(c.nb_v_token, c.page_size, c.head_dim) && kv8_apart(c.nb_v_head, c.n_head_kv, c.head_dim) &&
           kv8_apart(c.nb_s_page, c.n_pages, 4) && kv8_apart(c.nb_s_block, blocks, 4) && kv8_apart(c.nb_s_head, c.n_head_kv, 4);
}

static int kv8_rows_check(const q4k_kv8_rows *rows, bool store, bool &empty) {
    if (!rows || !rows->pages) return Q4K_EINVAL;
    const q4k_kv8_rows &a = *rows;
    const q4k_kv8_pages &c = *a.pages;
    if (!kv8_kind_ok(c)) return Q4K_EINVAL;
    if (a.type != Q4K_GGML_TYPE_F32 && a.type != Q4K_GGML_TYPE_F16 && a.type != Q4K_GGML_TYPE_BF16) return Q4K_EINVAL;
    const int st = kv8_tokens_check(a.n_tokens, a.n_requests, a.n_q, a.q_start, a.len, a.max_len, empty);
    if (st != Q4K_OK || empty) return st;
    const int es = a.type == Q4K_GGML_TYPE_F32 ? 4 : 2;
    if (store && (!a.k || !a.v)) return Q4K_EINVAL;
    if (!kv8_row_ok(a.k, a.nb_k_token, a.nb_k_head, es, c) || !kv8_row_ok(a.v, a.nb_v_token, a.nb_v_head, es, c)) return Q4K_EINVAL;
    if (!kv8_pages_ok(c, a.max_len, a.n_requests)) return Q4K_EINVAL;
    if (!kv8_pages_vec(c)) return Q4K_EUNSUPPORTED;
    if (store && !kv8_writable(c)) return Q4K_EINVAL;
    empty = !a.k && !a.v;
    return Q4K_OK;
}
static Kv8RowsParams kv8_rows_params(const q4k_kv8_rows &a) {
    Kv8RowsParams p{};
    p.c = kv8_cache(*a.pages);
    p.t = Kv8Tokens{a.q_start, a.len, (int)a.n_tokens, (int)a.n_requests, (int)a.n_q, (int)a.max_len};
    p.k = (char *)a.k;
    p.v = (char *)a.v;
    p.k_token = a.nb_k_token; p.k_head = a.nb_k_head; p.v_token = a.nb_v_token; p.v_head = a.nb_v_head;
    p.n_head = a.pages->n_head_kv;
    p.head_dim = a.pages->head_dim;
    return p;
}

using Kv8RowsFn = void (*)(Kv8RowsParams);
template <int THREADS, bool I8>
static Kv8RowsFn store_fn(int32_t type) {
    return type == Q4K_GGML_TYPE_F32 ? kv8_store_kernel<THREADS, I8, float>
           : type == Q4K_GGML_TYPE_F16 ? kv8_store_kernel<THREADS, I8, _Float16>
                                       : kv8_store_kernel<THREADS, I8, __bf16>;
}
template <bool I8>
static Kv8RowsFn load_fn(int32_t type) {
    return type == Q4K_GGML_TYPE_F32 ? kv8_load_kernel<I8, float>
           : type == Q4K_GGML_TYPE_F16 ? kv8_load_kernel<I8, _Float16>
                                       : kv8_load_kernel<I8, __bf16>;
}

}  // namespace q4k

using namespace q4k;

extern "C" {

int q4k_kv8_store(const q4k_kv8_rows *rows, void *stream) {
    bool empty;
    int st = kv8_rows_check(rows, true, empty);
    if (st != Q4K_OK || empty) return st;
    DeviceInfo *di;
    st = device_info(&di);
    if (st != Q4K_OK) return st;
    Kv8RowsParams p = kv8_rows_params(*rows);
    const int64_t block = rows->pages->block;
    p.blocks = (int)((rows->n_q + block - 2) / block + 1);
    const int64_t items = rows->n_requests * p.blocks;
    if (items > INT32_MAX / 2 / p.n_head) return Q4K_EUNSUPPORTED;
    const dim3 grid((unsigned)(items * p.n_head * 2));
    // A wave where a block's new rows fit its registers in two rounds, else four waves.
    const int64_t most = rows->n_q < block ? rows->n_q : block;
    const bool i8 = rows->pages->type == Q4K_TYPE_I8;
    if (most * p.head_dim <= 512) return launch(i8 ? store_fn<64, true>(rows->type) : store_fn<64, false>(rows->type), grid, 64, 0, stream, p);
    return launch(i8 ? store_fn<256, true>(rows->type) : store_fn<256, false>(rows->type), grid, 256, 0, stream, p);
}

int q4k_kv8_load(const q4k_kv8_rows *rows, void *stream) {
    bool empty;
    int st = kv8_rows_check(rows, false, empty);
    if (st != Q4K_OK || empty) return st;
    DeviceInfo *di;
    st = device_info(&di);
    if (st != Q4K_OK) return st;
    const Kv8RowsParams p = kv8_rows_params(*rows);
    const int64_t threads = (int64_t)p.head_dim / 8 * p.n_head;  // of a row, up to 2^36
    const int64_t n = rows->n_requests * rows->n_q;
    if (n > ((int64_t)INT32_MAX * 256 - 256) / threads) return Q4K_EUNSUPPORTED;
    const bool i8 = rows->pages->type == Q4K_TYPE_I8;
    return launch(i8 ? load_fn<true>(rows->type) : load_fn<false>(rows->type), dim3((unsigned)((n * threads + 255) / 256)), 256, 0, stream, p);
}

}  // extern "C"

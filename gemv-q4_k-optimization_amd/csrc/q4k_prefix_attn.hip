// q4k_prefix_attn.hip -- q4k_prefix_attn (include/q4k_batch.h): attention of a
// batch of requests over a prefix that they share and over their own tokens.
// The kernels are in q4k_attn.h; here are the argument checks, the split of the
// work and the launches.
#include "q4k_attn.h"

namespace q4k {

static bool pages_ok(const q4k_kv_pages &c, int64_t tokens, int64_t rows) {
    if (!c.k || !c.v || c.n_pages < 1 || c.n_pages > INT32_MAX || c.page_size < 1 || c.page_size > INT32_MAX) return false;
    if (!aligned(c.k, 2) || !aligned(c.v, 2) || !aligned(c.table, 4) || c.table_len < 0 || c.table_len > INT32_MAX) return false;
    if (c.table_len * c.page_size < tokens) return false;
    if (c.table ? rows > 1 && c.table_stride < 0 : c.table_len > c.n_pages / rows) return false;
    return true;
}
static bool pages_vec(const q4k_kv_pages &c) {
    return aligned(c.k, 16) && aligned(c.v, 16) &&
           ((c.nb_k_page | c.nb_k_token | c.nb_k_head | c.nb_v_page | c.nb_v_token | c.nb_v_head) & 15) == 0;
}

// Q4K_OK with empty set where there is nothing to do
static int attn_check(const q4k_prefix_attn_args *args, bool &empty) {
    if (!args) return Q4K_EINVAL;
    const q4k_prefix_attn_args &a = *args;
    empty = false;
    if (a.kv_type != Q4K_GGML_TYPE_F16 && a.kv_type != Q4K_GGML_TYPE_BF16) return Q4K_EINVAL;
    if (a.q_type != Q4K_GGML_TYPE_F32 && a.q_type != a.kv_type) return Q4K_EINVAL;
    if (a.n_head < 1 || a.n_head_kv < 1 || a.n_head % a.n_head_kv != 0 || a.head_dim < 1) return Q4K_EINVAL;
    if (a.n_tokens < 0 || a.n_requests < 0 || a.n_q < 0 || a.n_prefix < 0 || a.max_suffix < 0) return Q4K_EINVAL;
    if (a.n_tokens > INT32_MAX || a.n_requests > INT32_MAX || a.n_q > INT32_MAX || a.n_prefix > INT32_MAX ||
        a.max_suffix > INT32_MAX)
        return Q4K_EINVAL;
    if (!a.q_start && a.n_tokens != a.n_requests * a.n_q) return Q4K_EINVAL;
    if (a.n_tokens == 0 || a.n_requests == 0 || a.n_q == 0) {
        empty = true;
        return Q4K_OK;
    }
    const int es = a.q_type == Q4K_GGML_TYPE_F32 ? 4 : 2;
    if (!a.q || !a.dst || !aligned(a.q, es) || !aligned(a.dst, es) || !aligned(a.lse, 4) || !aligned(a.q_start, 4))
        return Q4K_EINVAL;
    if (a.nb_q_token % es != 0 || a.nb_q_head % es != 0 || a.nb_dst_token % es != 0 || a.nb_dst_head % es != 0)
        return Q4K_EINVAL;
    if ((a.n_head > 1 && (a.nb_q_head < es * (int64_t)a.head_dim || a.nb_dst_head < es * (int64_t)a.head_dim))) return Q4K_EINVAL;
    if (a.n_prefix > 0 && (!a.prefix || !pages_ok(*a.prefix, a.n_prefix, 1))) return Q4K_EINVAL;
    if (a.max_suffix > 0 &&
        (!a.suffix || !a.suffix_len || !aligned(a.suffix_len, 4) || !pages_ok(*a.suffix, a.max_suffix, a.n_requests)))
        return Q4K_EINVAL;
    if (a.head_dim % 8 != 0 || a.head_dim > Q4K_ATTN_MAX_HEAD_DIM) return Q4K_EUNSUPPORTED;
    if ((a.n_prefix > 0 && !pages_vec(*a.prefix)) || (a.max_suffix > 0 && !pages_vec(*a.suffix))) return Q4K_EUNSUPPORTED;
    if (a.n_requests * a.n_q > INT32_MAX || a.n_prefix > (1 << 30) || a.max_suffix > (1 << 30)) return Q4K_EUNSUPPORTED;
    return Q4K_OK;
}


static AttnCache attn_cache(const q4k_kv_pages &c, int64_t tokens) {
    AttnCache k{};
    k.k = (const char *)c.k;
    k.v = (const char *)c.v;
    k.k_page = c.nb_k_page; k.k_token = c.nb_k_token; k.k_head = c.nb_k_head;
    k.v_page = c.nb_v_page; k.v_token = c.nb_v_token; k.v_head = c.nb_v_head;
    k.table = c.table;
    k.table_stride = c.table_stride;
    k.n_pages = (int)c.n_pages;
    k.table_len = (int)c.table_len;
    k.one_page = !c.table && tokens <= c.page_size;
    k.page = fastdiv_init((uint32_t)c.page_size);
    return k;
}

static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

static int attn_plan(const q4k_prefix_attn_args &a, int cus, AttnPlan &pl) {
    pl = AttnPlan{};
    AttnParams &p = pl.p;
    if (a.n_prefix > 0) p.pre = attn_cache(*a.prefix, a.n_prefix);
    if (a.max_suffix > 0) p.suf = attn_cache(*a.suffix, a.max_suffix);
    p.q = (const char *)a.q;
    p.dst = (char *)a.dst;
    p.lse = a.lse;
    p.q_token = a.nb_q_token; p.q_head = a.nb_q_head; p.dst_token = a.nb_dst_token; p.dst_head = a.nb_dst_head;
    p.q_start = a.q_start;
    p.suffix_len = a.suffix_len;
    p.n_tokens = (int)a.n_tokens; p.n_requests = (int)a.n_requests; p.n_q = (int)a.n_q;
    p.n_prefix = (int)a.n_prefix; p.max_suffix = (int)a.max_suffix;
    p.n_head = a.n_head; p.n_head_kv = a.n_head_kv; p.group = a.n_head / a.n_head_kv; p.head_dim = a.head_dim;
    p.group_div = fastdiv_init((uint32_t)p.group);
    p.scale = a.scale;
    p.q_vec = aligned(a.q, 16) && (a.nb_q_token | a.nb_q_head) % 16 == 0;
    pl.dim = a.head_dim <= 64 ? 64 : a.head_dim <= 128 ? 128 : 256;
    if (a.n_tokens > INT32_MAX / p.group - 256) return Q4K_EUNSUPPORTED;
    const int64_t pre_rows = a.n_prefix > 0 ? a.n_tokens * p.group : 0, suf_rows = a.n_q * p.group;
    const int rows_of[3] = {16, pl.dim == 256 ? 16 : 32, pl.dim == 256 ? 64 : 128};
    // Streaming to this many rows of a KV head (prefix of 8 KV heads, us streaming /
    // sharing).  Each tile of 32 rows reads the positions again, so fewer where the
    // prefix's K and V are more than the caches hold, from 100 MB:
    //   128 dimensions, 16 bits: 96, then 32 (8192 positions: 64 rows 22.2 / 22.5, 128
    //   28.2 / 27.8, 256 39.5 / 34.4; 65536: 48 rows 80.6 / 69.5, 128 102 / 79);
    //   64 dimensions: 192, then 32 (8192: 192 rows 22.5 / 22.8, 384 33.8 / 31.3; 65536:
    //   128 rows 67.6 / 49.4);
    //   F32 queries on F16: 192, then 64 (8192: 192 rows 38.0 / 44.4, 512 88 / 78; 65536:
    //   64 rows 87.6 / 92.3, 128 119 / 104);
    //   256 dimensions, tiles of 16 rows: 32 (65536: 32 rows 131 / 152, 48 187 / 155);
    //   F32 queries on BF16, whose three terms a query leave sharing waves no registers:
    //   any, but for 256 dimensions (128 rows 109 / 89).
    const int terms = a.q_type != Q4K_GGML_TYPE_F32 ? 1 : a.kv_type == Q4K_GGML_TYPE_F16 ? 2 : 3;
    const bool far = (double)a.n_prefix * a.n_head_kv * pl.dim * 4 > 100e6;
    auto size_of = [&](int64_t rows, bool far) {
        const int64_t most = pl.dim == 256 ? 32 : terms == 3 ? INT32_MAX : far ? 32 * terms : terms == 1 && pl.dim == 128 ? 96 : 192;
        return rows <= 16 ? 0 : rows <= most ? 1 : 2;
    };
    pl.suf_size = size_of(suf_rows, false);
    pl.pre_size = a.n_prefix > 0 ? size_of(pre_rows, far) : pl.suf_size;
    if (pl.suf_size > pl.pre_size) pl.suf_size = pl.pre_size;  // (with q_start n_q may exceed the tokens there are)
    const int pr = rows_of[pl.pre_size], sr = rows_of[pl.suf_size];
    // Splits of one length for both parts, in whole steps of 128 positions: about
    // two workgroups per CU in all, however the positions are shared out.  Where
    // every workgroup streams, whose registers let two run on a CU, up to half as
    // much again if that makes them all run at once (16 requests of 32 heads behind
    // 8192 tokens: 26 us against 32 with 608 workgroups).
    const int64_t pt = a.n_prefix > 0 ? cdiv(pre_rows, pr) : 0, st = cdiv(suf_rows, sr);
    const bool own = a.max_suffix > 0 || a.n_prefix == 0;
    const int64_t per_pre = pt * a.n_head_kv, per_suf = own ? st * a.n_head_kv * a.n_requests : 0;
    if (per_pre > INT32_MAX / 4 || per_suf > INT32_MAX / 4) return Q4K_EUNSUPPORTED;
    const int64_t work = a.n_prefix * per_pre + a.max_suffix * per_suf;
    int64_t len = cdiv(cdiv(work, 2 * (int64_t)cus), 128) * 128;
    if (len < 128) len = 128;
    if (pl.pre_size < 2)
        for (int64_t l = len; l <= len * 3 / 2; l += cdiv(len, 16 * 128) * 128)
            if (per_pre * cdiv(a.n_prefix, l) + per_suf * cdiv(a.max_suffix, l) <= 2 * cus) {
                len = l;
                break;
            }
    if (len > (1 << 30)) len = 1 << 30;
    p.pre_len = p.suf_len = (int)len;
    if (a.n_prefix > 0) {
        p.pre_tiles = (int)pt;
        p.pre_splits = (int)cdiv(a.n_prefix, len);
        if (per_pre * p.pre_splits > INT32_MAX / 2) return Q4K_EUNSUPPORTED;
        p.pre_items = (int)(per_pre * p.pre_splits);
    }
    if (own) {
        p.suf_tiles = (int)st;
        p.suf_splits = a.max_suffix > 0 ? (int)cdiv(a.max_suffix, len) : 1;
        if (per_suf * p.suf_splits > INT32_MAX / 2) return Q4K_EUNSUPPORTED;
        p.suf_items = (int)(per_suf * p.suf_splits);
    }
    p.slots = p.pre_splits + p.suf_splits;
    // (the prefix's rows are all tokens: with q_start the join leaves those of no request out)
    p.join = p.slots > 1 || (a.n_prefix > 0 && a.q_start);
    // the join: four splits or so to a group of lanes, more rows to a workgroup where
    // that leaves groups (4096 rows of 2 splits: 8.5 us with a workgroup each)
    const int groups = 256 / (a.head_dim / 4);
    p.join_groups = 1;
    while (p.join_groups * 4 < p.slots && p.join_groups * 2 <= groups) p.join_groups *= 2;
    p.join_rows = groups / p.join_groups;
    if (p.join) {
        const int64_t rows = a.n_tokens * a.n_head;
        if (rows > ((int64_t)1 << 50) / p.slots / (a.head_dim + 2)) return Q4K_EUNSUPPORTED;
        pl.bytes = (size_t)(rows * p.slots * (a.head_dim + 2) * 4);
    }
    // (the join counts its rows in 31 bits, up to a workgroup's past the last one)
    if (a.n_requests * a.n_q > (INT32_MAX - 256) / a.n_head) return Q4K_EUNSUPPORTED;
    const bool f32 = a.q_type == Q4K_GGML_TYPE_F32;
    if (a.kv_type == Q4K_GGML_TYPE_F16) f32 ? attn_kernel_f16_f32(pl) : attn_kernel_f16(pl);
    else f32 ? attn_kernel_bf16_f32(pl) : attn_kernel_bf16(pl);
    return Q4K_OK;
}

}  // namespace q4k

using namespace q4k;

extern "C" {

size_t q4k_prefix_attn_workspace_bytes(const q4k_prefix_attn_args *args) {
    bool empty;
    if (attn_check(args, empty) != Q4K_OK || empty) return 0;
    DeviceInfo *di;
    AttnPlan pl;
    if (device_info(&di) != Q4K_OK || attn_plan(*args, di->cus, pl) != Q4K_OK) return 0;
    return pl.bytes;
}

int q4k_prefix_attn(const q4k_prefix_attn_args *args, void *workspace, size_t workspace_bytes, void *stream) {
    bool empty;
    int st = attn_check(args, empty);
    if (st != Q4K_OK || empty) return st;
    DeviceInfo *di;
    st = device_info(&di);
    if (st != Q4K_OK) return st;
    AttnPlan pl;
    st = attn_plan(*args, di->cus, pl);
    if (st != Q4K_OK) return st;
    st = ensure_lds(di, pl.kernel, pl.lds);
    if (st != Q4K_OK) return st;
    Workspace ws;
    st = ws.begin(workspace, workspace_bytes, pl.bytes, stream);
    if (st != Q4K_OK) return st;
    AttnParams &p = pl.p;
    p.part_o = (float *)ws.ptr;
    p.part_ml = (float2 *)(p.part_o + (int64_t)p.n_tokens * p.n_head * p.slots * p.head_dim);
    using Fn = void (*)(AttnParams);
    st = launch((Fn)pl.kernel, dim3((unsigned)(p.pre_items + p.suf_items)), 256, pl.lds, stream, p);
    if (st == Q4K_OK && p.join) {
        const bool f32 = args->q_type == Q4K_GGML_TYPE_F32, f16 = args->kv_type == Q4K_GGML_TYPE_F16;
        Fn join = f32 ? prefix_attn_join_kernel<float> : f16 ? prefix_attn_join_kernel<_Float16> : prefix_attn_join_kernel<__bf16>;
        st = launch(join, dim3((unsigned)cdiv((int64_t)p.n_requests * p.n_q * p.n_head, p.join_rows)), 256, 0, stream, p);
    }
    return ws.end(st, stream);
}

}  // extern "C"

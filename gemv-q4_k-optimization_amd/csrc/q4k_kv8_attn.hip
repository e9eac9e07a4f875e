// q4k_kv8_attn.hip -- q4k_kv8_attn (include/q4k_step.h): attention of a batch of
// requests over their paged caches of 8 bits.  The kernel is in q4k_kv8_attn.h;
// here are the argument checks, the split of the work and the launches.
#include "q4k_kv8_attn.h"

namespace q4k {

static int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

static int kv8_attn_check(const q4k_kv8_attn_args *args, bool &empty) {
    if (!args || !args->pages) return Q4K_EINVAL;
    const q4k_kv8_attn_args &a = *args;
    const q4k_kv8_pages &c = *a.pages;
    if (!kv8_kind_ok(c)) return Q4K_EINVAL;
    if (a.q_type != Q4K_GGML_TYPE_F32 && a.q_type != Q4K_GGML_TYPE_F16 && a.q_type != Q4K_GGML_TYPE_BF16) return Q4K_EINVAL;
    if (a.n_head < 1 || a.n_head % c.n_head_kv != 0) return Q4K_EINVAL;
    const int st = kv8_tokens_check(a.n_tokens, a.n_requests, a.n_q, a.q_start, a.len, a.max_len, empty);
    if (st != Q4K_OK || empty) return st;
    const int es = a.q_type == Q4K_GGML_TYPE_F32 ? 4 : 2;
    if (!a.q || !a.dst || !aligned(a.q, es) || !aligned(a.dst, es) || !aligned(a.lse, 4)) return Q4K_EINVAL;
    if ((a.nb_q_token | a.nb_q_head | a.nb_dst_token | a.nb_dst_head) & (es - 1)) return Q4K_EINVAL;
    if (a.n_head > 1 && (a.nb_q_head < es * (int64_t)c.head_dim || a.nb_dst_head < es * (int64_t)c.head_dim)) return Q4K_EINVAL;
    if (!kv8_pages_ok(c, a.max_len, a.n_requests)) return Q4K_EINVAL;
    return kv8_pages_vec(c) ? Q4K_OK : Q4K_EUNSUPPORTED;
}

static int kv8_attn_plan(const q4k_kv8_attn_args &a, int cus, Kv8AttnPlan &pl) {
    pl = Kv8AttnPlan{};
    const q4k_kv8_pages &c = *a.pages;
    AttnParams &p = pl.p.a;
    pl.p.c = kv8_cache(c);
    p.q = (const char *)a.q;
    p.dst = (char *)a.dst;
    p.lse = a.lse;
    p.q_token = a.nb_q_token; p.q_head = a.nb_q_head; p.dst_token = a.nb_dst_token; p.dst_head = a.nb_dst_head;
    p.q_start = a.q_start;
    p.suffix_len = a.len;
    p.n_tokens = (int)a.n_tokens; p.n_requests = (int)a.n_requests; p.n_q = (int)a.n_q;
    p.max_suffix = (int)a.max_len;
    p.n_head = a.n_head; p.n_head_kv = c.n_head_kv; p.group = a.n_head / c.n_head_kv; p.head_dim = c.head_dim;
    p.group_div = fastdiv_init((uint32_t)p.group);
    p.scale = a.scale;
    p.q_vec = aligned(a.q, 16) && ((a.nb_q_token | a.nb_q_head) & 15) == 0;
    pl.dim = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
    pl.i8 = c.type == Q4K_TYPE_I8;
    pl.block8 = c.block % 8 == 0;
    if (a.n_q > INT32_MAX / p.group - 256) return Q4K_EUNSUPPORTED;
    const int64_t rows = a.n_q * p.group;
    pl.rt = rows <= 16 || pl.dim == 256 ? 1 : 2;
    const int64_t tiles = cdiv(rows, 16 * pl.rt);
    if (tiles > INT32_MAX / 4 / p.n_head_kv / a.n_requests) return Q4K_EUNSUPPORTED;
    const int64_t per = tiles * p.n_head_kv * a.n_requests;
    p.suf_tiles = (int)tiles;
    a.q_type == Q4K_GGML_TYPE_F32 ? kv8_attn_f32(pl) : a.q_type == Q4K_GGML_TYPE_F16 ? kv8_attn_f16(pl) : kv8_attn_bf16(pl);
    const int64_t steps = cdiv(a.max_len, kKv8Step), most = (int64_t)pl.wgs * cus;
    // (the steps of one request are counted in 31 bits)
    if (steps > INT32_MAX / p.n_head_kv / tiles) return Q4K_EUNSUPPORTED;
    int64_t each = cdiv(per * steps, most);
    if (each < kKv8Least) each = kKv8Least;
    int64_t slots = 0;  // of parts
    if (each > kKv8Few) {
        pl.p.shares = (int)most;
        pl.kernel = pl.dealt;
        pl.lds += kKv8Deal;
        pl.start_bytes = ((size_t)a.n_requests * 8 + 8 + 15) / 16 * 16;
        slots = 2 * most;
        p.suf_items = (int)most;
    } else {
        pl.p.each = (int)each;
        const int64_t parts = steps > each ? cdiv(steps, each) : 1;
        p.suf_items = (int)(per * parts);
        if (parts > 1) slots = p.suf_items;
    }
    if (slots) {
        // (parts of a row; dealt out: of a request twice as long as the others)
        const JoinSplit join = join_split(p.head_dim, pl.p.shares ? 2 * most / per + 1 : slots / per);
        p.join_groups = join.groups;
        p.join_rows = join.rows;
        pl.bytes = pl.start_bytes + (size_t)slots * 16 * pl.rt * (p.head_dim + 2) * 4;
    }
    pl.slots = slots;
    // (the join counts its rows in 31 bits, up to a workgroup's past the last one)
    if (a.n_requests * a.n_q > (INT32_MAX - 256) / a.n_head) return Q4K_EUNSUPPORTED;
    if (!launches(p.suf_items, 256) || (slots && !launches(cdiv(a.n_requests * a.n_q * a.n_head, p.join_rows), kJoinThreads))) return Q4K_EUNSUPPORTED;
    return Q4K_OK;
}

}  // namespace q4k

using namespace q4k;

extern "C" {

size_t q4k_kv8_attn_workspace_bytes(const q4k_kv8_attn_args *args) {
    bool empty;
    if (kv8_attn_check(args, empty) != Q4K_OK || empty) return 0;
    DeviceInfo *di;
    Kv8AttnPlan pl;
    if (device_info(&di) != Q4K_OK || kv8_attn_plan(*args, di->cus, pl) != Q4K_OK) return 0;
    return pl.bytes;
}

int q4k_kv8_attn(const q4k_kv8_attn_args *args, void *workspace, size_t workspace_bytes, void *stream) {
    bool empty;
    int st = kv8_attn_check(args, empty);
    if (st != Q4K_OK || empty) return st;
    DeviceInfo *di;
    st = device_info(&di);
    if (st != Q4K_OK) return st;
    Kv8AttnPlan pl;
    st = kv8_attn_plan(*args, di->cus, pl);
    if (st != Q4K_OK) return st;
    st = ensure_lds(di, pl.kernel, pl.lds);
    if (st != Q4K_OK) return st;
    Workspace ws;
    st = ws.begin(workspace, workspace_bytes, pl.bytes, stream);
    if (st != Q4K_OK) return st;
    AttnParams &p = pl.p.a;
    pl.p.starts = (double *)ws.ptr;
    p.part_o = (float *)((char *)ws.ptr + pl.start_bytes);
    p.part_ml = (float2 *)(p.part_o + pl.slots * 16 * pl.rt * p.head_dim);
    st = launch((void (*)(Kv8AttnParams))pl.kernel, dim3((unsigned)p.suf_items), 256, pl.lds, stream, pl.p);
    if (st == Q4K_OK && pl.slots) {
        const int64_t rows = (int64_t)p.n_requests * p.n_q * p.n_head;
        st = launch((void (*)(Kv8AttnParams))pl.join, dim3((unsigned)cdiv(rows, p.join_rows)), 256, 0, stream, pl.p);
    }
    return ws.end(st, stream);
}

}  // extern "C"

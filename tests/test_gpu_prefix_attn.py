"""q4k_prefix_attn against 64 bits: prefixes and suffixes of zero, one and many
tokens, several queries a request, head layouts, pages that end inside a tile,
strides, unseen values of any kind, rows that see nothing."""
import pytest
import torch

import _batch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


class Case:
    """A batch with its caches; memory that no query may see holds NaN."""

    def __init__(self, gpu, B, nq, H, hk, D, prefix, suffix, page, qt=F32, kv=F16, seed=0, lens=None, spans=None, prefix_page=None, order=True):
        g = torch.Generator(device=gpu).manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, device=gpu, generator=g)  # noqa: E731
        self.B, self.nq, self.D, self.n_prefix, self.most = B, nq, D, prefix, suffix
        self.spans = spans or [(r * nq, r * nq + nq) for r in range(B)]
        self.q = rnd(self.spans[-1][1] if B else 0, H, D).to(qt)
        self.q_start = torch.tensor([0] + [s[1] for s in self.spans], dtype=torch.int32, device=gpu) if spans else None
        self.prefix = self.suffix = None
        if prefix:
            pp = prefix_page or prefix
            n = -(-prefix // pp)
            k, v = self.pool(rnd, n + 1, pp, hk, D, kv)
            self.pt = torch.randperm(n, device=gpu, generator=g).int() if prefix_page else torch.zeros(1, dtype=torch.int32, device=gpu)
            self.fill(rnd, k, v, self.pt, prefix)
            self.prefix = (k, v, self.pt)
        self.lens = None
        if suffix:
            per = -(-suffix // page)
            k, v = self.pool(rnd, B * per + 2, page, hk, D, kv)
            self.st = torch.randperm(B * per + 2, device=gpu, generator=g)[:B * per].view(B, per).int().contiguous()
            self.lens = lens if lens is not None else torch.randint(0, suffix + 1, (B,), device=gpu, generator=g).tolist()
            for r in range(B):
                self.fill(rnd, k, v, self.st[r], self.lens[r])
            self.suffix = (k, v, self.st)
        self.scale = D ** -0.5

    @staticmethod
    def pool(rnd, n, page, hk, D, kv):
        return [torch.full((n, page, hk, D), float("nan"), dtype=kv, device=rnd(1).device) for _ in range(2)]

    @staticmethod
    def fill(rnd, k, v, table, length):
        page = k.shape[1]
        for i in range(-(-length // page)):
            n = min(page, length - i * page)
            for t in (k, v):
                t[int(table[i]), :n] = rnd(n, *t.shape[2:]).to(t.dtype)

    def run(self, Q, **kw):
        pre = Q.KVPages(*self.prefix[:2], table=self.prefix[2]) if self.prefix else None
        suf = Q.KVPages(*self.suffix[:2], table=self.suffix[2]) if self.suffix else None
        lens = torch.tensor(self.lens, dtype=torch.int32, device=self.q.device) if self.suffix else None
        lse = torch.full(self.q.shape[:2], 7.0, device=self.q.device)
        out = Q.prefix_attention(self.q, pre, self.n_prefix, suf, lens, self.most, n_q=self.nq, q_start=self.q_start, scale=self.scale,
                                 lse=lse, **kw)
        return out, lse

    def check(self, Q, **kw):
        out, lse = self.run(Q, **kw)
        want, wl, tol, tl = _batch.attention(self.q, self.spans, self.prefix, self.suffix, (self.n_prefix, self.lens), self.scale)
        a = _batch.assert_close(out, want, tol, "out")
        b = _batch.assert_close(lse, wl, tl, "lse")
        return out, lse, max(a, b)


TYPES = [(F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("B,nq,H,hk,D,prefix,suffix,page", [
    (1, 1, 1, 1, 8, 1, 0, 16), (1, 1, 4, 2, 64, 0, 1, 16), (2, 1, 8, 8, 128, 33, 20, 16), (3, 1, 32, 8, 128, 500, 70, 16),
    (5, 1, 28, 4, 80, 129, 100, 48), (4, 1, 8, 1, 256, 200, 33, 32), (2, 5, 24, 8, 64, 257, 61, 24), (7, 3, 6, 2, 96, 64, 40, 7),
    (17, 1, 16, 2, 128, 300, 90, 100), (40, 2, 14, 2, 64, 1000, 30, 16), (70, 1, 8, 1, 128, 2100, 65, 64), (3, 40, 4, 2, 40, 190, 300, 64),
    (1, 1, 8, 8, 128, 9000, 5, 16), (2, 1, 4, 1, 128, 0, 3000, 48), (33, 1, 64, 8, 128, 700, 128, 32)])
def test_attention_sizes(Q, gpu, qt, kv, B, nq, H, hk, D, prefix, suffix, page):
    Case(gpu, B, nq, H, hk, D, prefix, suffix, page, qt, kv, seed=B + D).check(Q)


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("B,nq,H,hk,D,prefix,suffix,page", [
    (2, 150, 2, 1, 128, 100, 260, 16), (2, 130, 4, 1, 64, 70, 200, 40), (1, 60, 4, 2, 256, 65, 90, 16), (3, 100, 3, 1, 96, 0, 130, 16)])
def test_attention_many_queries_a_request(Q, gpu, qt, kv, B, nq, H, hk, D, prefix, suffix, page):
    """Rows enough that waves share the suffix too, whose bound is the queries' own."""
    c = Case(gpu, B, nq, H, hk, D, prefix, suffix, page, qt, kv, seed=D, lens=[suffix, nq + 3, nq // 2][:B])
    want = c.run(Q)
    c.check(Q)
    # what only the last query sees leaves the others alone
    k, v, t = c.suffix
    for r, length in enumerate(c.lens):
        j = length - 1
        v[int(t[r, j // page]), j % page, :, ::2] = float("-inf")
        k[int(t[r, j // page]), j % page] = float("nan")
    got = c.run(Q)
    for r in range(B):
        lo, hi = r * nq, (r + 1) * nq - 1
        assert torch.equal(got[0][lo:hi], want[0][lo:hi]) and torch.equal(got[1][lo:hi], want[1][lo:hi])
        assert not torch.isfinite(got[0][hi].float()).any()
    # an infinite value that several queries see, behind the bound of the others
    c = Case(gpu, B, nq, H, hk, D, prefix, suffix, page, qt, kv, seed=D, lens=[suffix, nq + 3, nq // 2][:B])
    k, v, t = c.suffix
    j = c.lens[0] - 5
    v[int(t[0, j // page]), j % page, :, 1] = float("inf")
    c.check(Q)


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("B,nq,H,hk,D,prefix,suffix,page", [(35, 1, 4, 4, 256, 33, 70, 16), (12, 6, 8, 2, 128, 300, 70, 16)])
def test_attention_shared_prefix_streamed_suffix(Q, gpu, qt, kv, B, nq, H, hk, D, prefix, suffix, page):
    Case(gpu, B, nq, H, hk, D, prefix, suffix, page, qt, kv, seed=B).check(Q)


@pytest.mark.parametrize("qt,kv,B,nq,H,hk,D,prefix,suffix", [
    (F16, F16, 1, 5, 64, 8, 128, 25100, 40), (F32, F16, 2, 1, 280, 8, 64, 50100, 20)])
def test_attention_few_rows_over_a_large_prefix(Q, gpu, qt, kv, B, nq, H, hk, D, prefix, suffix):
    """More than 100 MB of keys and values, whose tiles waves share from few rows on."""
    Case(gpu, B, nq, H, hk, D, prefix, suffix, 16, qt, kv, seed=B).check(Q)


@pytest.mark.parametrize("qt,kv", TYPES[:1] + TYPES[3:])
@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129])
def test_attention_lengths_around_a_tile(Q, gpu, qt, kv, prefix):
    n = 6
    Case(gpu, n, 1, 8, 2, 128, prefix, 130, 16, qt, kv, seed=prefix, lens=[0, 1, 64, 65, 129, 130]).check(Q)


@pytest.mark.parametrize("kv", [F16, BF16])
def test_attention_rows_that_see_nothing(Q, gpu, kv):
    """No prefix: an empty request, and queries before its first own token."""
    c = Case(gpu, 4, 3, 8, 2, 64, 0, 40, 16, F32, kv, lens=[0, 1, 2, 40])
    out, lse, _ = c.check(Q)
    assert not out[:3].any() and (lse[:3] == -float("inf")).all()
    assert not out[3:5].any() and lse[5].isfinite().all()
    c = Case(gpu, 3, 1, 4, 4, 64, 0, 0, 16, F32, kv)
    k = torch.full((1, 4, 4, 64), float("nan"), dtype=kv, device=gpu)
    got = Q.prefix_attention(c.q, Q.KVPages(k, k), 0)
    assert not got.any()


@pytest.mark.parametrize("qt,kv", TYPES)
def test_attention_queries_of_their_own_number(Q, gpu, qt, kv):
    spans = [(0, 3), (3, 3), (3, 4), (4, 11), (11, 12)]
    Case(gpu, 5, 7, 12, 4, 64, 77, 50, 16, qt, kv, lens=[10, 4, 0, 50, 33], spans=spans).check(Q)


@pytest.mark.parametrize("qt,kv", TYPES)
def test_attention_pages_of_the_prefix(Q, gpu, qt, kv):
    for page in (1, 5, 16, 40, 200):
        Case(gpu, 9, 1, 16, 4, 128, 333, 20, 16, qt, kv, prefix_page=page).check(Q)


def test_attention_pages_out_of_range_are_not_seen(Q, gpu):
    c = Case(gpu, 3, 1, 8, 2, 128, 200, 100, 16, F32, F16, lens=[100, 50, 33], prefix_page=20)
    c.pt[3] = -1
    c.pt[7] = 10 ** 6
    c.st[0, 2] = -5
    c.st[1, 0] = 2 ** 31 - 1
    c.check(Q)
    c.pt.fill_(-1)
    c.st.fill_(-1)
    out, lse = c.run(Q)
    assert not out.any() and (lse == -float("inf")).all()


def test_attention_lengths_beyond_the_bound_are_clamped(Q, gpu):
    c = Case(gpu, 3, 1, 8, 2, 64, 30, 48, 16, F16, F16, lens=[48, 48, 0])
    want = c.run(Q)
    c.lens = [100, 2 ** 31 - 1, -7]
    got = c.run(Q)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("qt,kv", TYPES)
def test_attention_infinite_values_behind_the_causal_bound(Q, gpu, qt, kv):
    """A later token's values and keys of inf or NaN leave earlier queries alone."""
    c = Case(gpu, 2, 4, 8, 2, 64, 50, 40, 16, qt, kv, lens=[40, 17])
    want = c.run(Q)
    k, v, t = c.suffix
    for r, length in enumerate(c.lens):
        j = length - 1
        v[int(t[r, j // 16]), j % 16] = float("inf")
        k[int(t[r, j // 16]), j % 16] = float("nan")
    got = c.run(Q)
    for r in range(2):
        assert torch.equal(got[0][4 * r:4 * r + 3], want[0][4 * r:4 * r + 3])
        assert torch.equal(got[1][4 * r:4 * r + 3], want[1][4 * r:4 * r + 3])
        assert not torch.isfinite(got[0][4 * r + 3].float()).any()


@pytest.mark.parametrize("qt,kv", TYPES)
def test_attention_peaked_flat_and_large_scores(Q, gpu, qt, kv):
    c = Case(gpu, 6, 1, 8, 2, 128, 700, 60, 16, qt, kv, seed=3)
    c.q[0] = 0                    # flat
    c.q[1] = c.q[1] * 30          # one position takes all
    c.prefix[0][0, 690] = c.prefix[0][0, 690] * 20   # the maximum comes late
    c.q[2] = c.q[2] * 1e-3
    c.check(Q)
    c.scale = -1.5
    c.check(Q)
    c.scale = 0.0
    c.check(Q)


def test_attention_f32_queries_of_any_magnitude(Q, gpu):
    """F32 queries outside F16's range: the row is scaled by a power of two."""
    c = Case(gpu, 4, 1, 8, 2, 64, 300, 20, 16, F32, F16, seed=5)
    base = c.q.clone()
    for e in (1e9, 1e-9):
        c.q, c.scale = base * e, 64 ** -0.5 / e
        c.check(Q)


@pytest.mark.parametrize("qt,kv", TYPES)
def test_attention_strides(Q, gpu, qt, kv):
    """Heads before tokens, rows apart, outputs between other values."""
    c = Case(gpu, 5, 2, 12, 4, 64, 90, 40, 16, qt, kv, seed=8)
    want = c.run(Q)
    nan = float("nan")
    for which in ("prefix", "suffix"):
        k, v, t = getattr(c, which)
        k2 = torch.full((k.shape[0], 4, k.shape[1] + 1, 72), nan, dtype=kv, device=gpu).permute(0, 2, 1, 3)[:, :-1, :, :64]
        v2 = torch.full((k.shape[0], k.shape[1], 5, 64), nan, dtype=kv, device=gpu)[:, :, 1:]
        k2.copy_(k)
        v2.copy_(v)
        setattr(c, which, (k2, v2, t))
    q2 = torch.full((10, 13, 67), nan, dtype=qt, device=gpu)[:, :12, 3:]
    q2.copy_(c.q)
    c.q = q2
    big = torch.full((12, 10, 69), nan, dtype=qt, device=gpu)
    out = big.permute(1, 0, 2)[:, :, 1:65]
    got = c.run(Q, out=out)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.isnan(big).sum() == big.numel() - out.numel()


def test_attention_cache_past_32_bits(Q, gpu):
    """Pages and tokens more than 4 GiB into the cache."""
    D, hk, page = 64, 2, 16
    stride = (1 << 31) + 64
    big = torch.zeros(stride + 2 * page * hk * D + 64, dtype=F16, device=gpu)
    pool = big.as_strided((2, page, hk, D), (stride, hk * D, D, 1))
    c = Case(gpu, 2, 1, 4, hk, D, 30, 16, page, F32, F16, prefix_page=page, lens=[16, 3])
    k, v, t = c.prefix
    pool.copy_(k[t.long()])
    c.prefix = (pool, v[t.long()], torch.arange(2, dtype=torch.int32, device=gpu))
    c.check(Q)
    # a contiguous prefix with far tokens
    far = (1 << 28) + 8
    big = torch.zeros(16 * far + 2 * D, dtype=F16, device=gpu)
    pool = big.as_strided((1, 17, hk, D), (0, far, D, 1))
    c = Case(gpu, 2, 1, 4, hk, D, 17, 16, page, F32, F16, lens=[16, 3])
    pool.copy_(c.prefix[0][:1])
    c.prefix = (pool, c.prefix[1][:1], c.pt)
    c.check(Q)


def test_attention_repeated_bits_and_workspace(Q, gpu):
    c = Case(gpu, 16, 1, 32, 8, 128, 3000, 100, 16, F32, F16)
    want = c.run(Q)
    pre, suf = Q.KVPages(*c.prefix[:2], table=c.prefix[2]), Q.KVPages(*c.suffix[:2], table=c.suffix[2])
    lens = torch.tensor(c.lens, dtype=torch.int32, device=gpu)
    ws = Q.prefix_attention_workspace(c.q, pre, 3000, suf, lens, 100)
    ws.fill_(255)
    for _ in range(3):
        got = c.run(Q, workspace=ws)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if ws.numel() > 16:
        with pytest.raises(Q.Q4KError):
            c.run(Q, workspace=ws[:16])


def test_attention_without_tables(Q, gpu):
    c = Case(gpu, 4, 1, 8, 2, 64, 100, 33, 48, F16, F16, seed=4)
    want = c.run(Q)
    k, v, t = c.suffix
    at = t.long()[:, 0]
    lens = torch.tensor(c.lens, dtype=torch.int32, device=gpu)
    got = Q.prefix_attention(c.q, Q.KVPages(*(x[:1] for x in c.prefix[:2])), 100, Q.KVPages(k[at], v[at]), lens, 33, scale=c.scale)
    assert torch.equal(got, want[0])


def test_attention_graph_and_stream(Q, gpu):
    """A captured call follows lengths, tables and queries that change between replays."""
    c = Case(gpu, 6, 1, 8, 2, 128, 900, 200, 16, F32, F16, lens=[200] * 6)
    pre, suf = Q.KVPages(*c.prefix[:2], table=c.prefix[2]), Q.KVPages(*c.suffix[:2], table=c.suffix[2])
    lens = torch.full((6,), 200, dtype=torch.int32, device=gpu)
    out, lse = torch.empty_like(c.q), torch.empty(6, 8, device=gpu)
    ws = Q.prefix_attention_workspace(c.q, pre, 900, suf, lens, 200)
    call = lambda **kw: Q.prefix_attention(c.q, pre, 900, suf, lens, 200, lse=lse, **kw)  # noqa: E731
    call(out=out, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out=out, workspace=ws)
    for rep in range(4):
        c.q.normal_()
        lens.copy_(torch.randint(0, 201, (6,), device=gpu))
        c.st.copy_(c.st.roll(1, 0))
        graph.replay()
        torch.cuda.synchronize()
        l1 = lse.clone()
        assert torch.equal(out, call()) and torch.equal(l1, lse), rep
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = call(stream=s)
    s.synchronize()
    assert torch.equal(got, out)


def test_attention_refusals_of_the_binding(Q, gpu):
    c = Case(gpu, 2, 1, 8, 2, 64, 30, 20, 16, F16, F16)
    pre, suf = Q.KVPages(*c.prefix[:2], table=c.prefix[2]), Q.KVPages(*c.suffix[:2], table=c.suffix[2])
    lens = torch.tensor([20, 20], dtype=torch.int32, device=gpu)
    for bad in (lambda: Q.prefix_attention(c.q.bfloat16(), pre, 30, suf, lens, 20), ):
        with pytest.raises(Q.Q4KError):
            bad()
    for bad in (lambda: Q.prefix_attention(c.q, pre, 30, suf, lens.long(), 20), lambda: Q.prefix_attention(c.q, pre, 30, suf, lens[:1], 20),
                lambda: Q.prefix_attention(c.q[:, :, :32], pre, 30), lambda: Q.KVPages(c.prefix[0], c.prefix[1].bfloat16()),
                lambda: Q.KVPages(*c.prefix[:2], table=c.pt.long()), lambda: Q.prefix_attention(c.q, None, 30, suf, lens, 20)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(Q.Q4KError):
        Q.prefix_attention(c.q, pre, 61)


def test_attention_refuses_operands_in_host_memory(Q, gpu):
    c = Case(gpu, 2, 1, 8, 2, 64, 3000, 20, 16, F16, F16)
    pre, suf = Q.KVPages(*c.prefix[:2], table=c.prefix[2]), Q.KVPages(*c.suffix[:2], table=c.suffix[2])
    lens = torch.tensor(c.lens, dtype=torch.int32, device=gpu)
    ws = Q.prefix_attention_workspace(c.q, pre, 3000, suf, lens, 20)
    for bad in (dict(workspace=ws.cpu()), dict(workspace=ws[:1].expand(ws.numel())), dict(out=torch.empty_like(c.q, device="cpu"))):
        with pytest.raises(ValueError):
            Q.prefix_attention(c.q, pre, 3000, suf, lens, 20, **bad)
    with pytest.raises(ValueError):
        Q.prefix_attention(c.q.cpu(), pre, 3000, suf, lens, 20)
    with pytest.raises(ValueError):
        Q.prefix_attention(c.q, pre, 3000, suf, lens.cpu(), 20)


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("heads,prefix,suffix", [(4, 1, 0), (4, 100, 0), (4, 3000, 0), (64, 120, 0), (64, 3000, 0), (4, 100, 40), (64, 0, 40)])
def test_attention_leaves_tokens_of_no_request_alone(Q, gpu, qt, kv, heads, prefix, suffix):
    """Tokens before the first request, past the n_q of a request and behind the last one."""
    c = Case(gpu, 4, 3, heads, 2, 64, prefix, suffix, 16, qt, kv, seed=heads)
    spans, n = [(2, 4), (4, 4), (4, 7), (9, 10)], 13    # the third request has 5 tokens, of which 3 count
    starts = torch.tensor([2, 4, 4, 9, 10], dtype=torch.int32, device=gpu)
    c.q = torch.randn(n, heads, 64, device=gpu).to(qt)
    pre = Q.KVPages(*c.prefix[:2]) if prefix else None
    suf = Q.KVPages(*c.suffix[:2], table=c.suffix[2]) if suffix else None
    lens = torch.tensor(c.lens, dtype=torch.int32, device=gpu) if suffix else None
    out, lse = torch.full_like(c.q, 7.0), torch.full((n, heads), 7.0, device=gpu)
    Q.prefix_attention(c.q, pre, prefix, suf, lens, suffix, n_q=3, q_start=starts, scale=c.scale, out=out, lse=lse)
    # (a prefix of its own page, so that its table is the pages in order)
    want, wl, tol, tl = _batch.attention(c.q, spans, c.prefix, c.suffix, (prefix, c.lens), c.scale)
    mine = torch.zeros(n, dtype=torch.bool)
    for lo, hi in spans:
        mine[lo:hi] = True
    _batch.assert_close(out.cpu()[mine], want[mine], tol[mine], "out")
    _batch.assert_close(lse.cpu()[mine], wl[mine], tl[mine], "lse")
    assert (out.cpu()[~mine] == 7).all() and (lse.cpu()[~mine] == 7).all()


def test_attention_keeps_the_description_of_a_cache(Q, gpu):
    """One KVPages without a table as the requests' pages of batches of several
    sizes, then as a prefix, and as both in one call."""
    g = torch.Generator(device=gpu).manual_seed(2)
    k, v = (torch.randn(12, 16, 2, 64, device=gpu, generator=g).half() for _ in range(2))
    q = torch.randn(4, 8, 64, device=gpu, generator=g).half()
    lens = torch.tensor([16, 9, 3, 30], dtype=torch.int32, device=gpu)
    pool, scale = Q.KVPages(k, v), 64 ** -0.5
    table = lambda n: torch.arange(12 // n * n, dtype=torch.int32, device=gpu).view(n, -1)  # noqa: E731

    def check(n, n_prefix, most):
        got = Q.prefix_attention(q[:n], pool if n_prefix else None, n_prefix, pool if most else None, lens[:n] if most else None, most)
        cache = (k, v, torch.arange(12))
        want, _, tol, _ = _batch.attention(q[:n], [(i, i + 1) for i in range(n)], cache if n_prefix else None, (k, v, table(n)) if most else None,
                                           (n_prefix, lens[:n].tolist() if most else None), scale)
        _batch.assert_close(got, want, tol, f"{n} requests, {n_prefix} + {most}")

    for n, n_prefix, most in ((4, 0, 40), (2, 0, 90), (3, 180, 0), (4, 180, 40), (1, 192, 16)):
        check(n, n_prefix, most)


@pytest.mark.parametrize("qt,kv", TYPES)
def test_attention_without_a_bound_on_the_queries_takes_all(Q, gpu, qt, kv):
    spans = [(0, 3), (3, 3), (3, 4), (4, 11), (11, 12)]
    c = Case(gpu, 5, 7, 12, 4, 64, 77, 50, 16, qt, kv, lens=[10, 4, 0, 50, 33], spans=spans)
    pre, suf = Q.KVPages(*c.prefix[:2], table=c.prefix[2]), Q.KVPages(*c.suffix[:2], table=c.suffix[2])
    lens = torch.tensor(c.lens, dtype=torch.int32, device=gpu)
    ws = Q.prefix_attention_workspace(c.q, pre, 77, suf, lens, 50, q_start=c.q_start)
    out = torch.full_like(c.q, 7.0)
    Q.prefix_attention(c.q, pre, 77, suf, lens, 50, q_start=c.q_start, scale=c.scale, out=out, workspace=ws)
    want, _, tol, _ = _batch.attention(c.q, spans, c.prefix, c.suffix, (77, c.lens), c.scale)
    _batch.assert_close(out, want, tol, "out")


def test_attention_refuses_a_table_without_rows(Q, gpu):
    """A table of no requests for one request, whose pages would be taken in order instead."""
    c = Case(gpu, 1, 1, 8, 2, 64, 30, 20, 16, F16, F16, lens=[20])
    pre, lens = Q.KVPages(*c.prefix[:2], table=c.prefix[2]), torch.tensor([20], dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError):
        Q.prefix_attention(c.q, pre, 30, Q.KVPages(*c.suffix[:2], table=c.st[:0]), lens, 20)
    with pytest.raises(ValueError):
        Q.prefix_attention(c.q, Q.KVPages(*c.prefix[:2], table=c.st[:0]), 30)
    assert Q.prefix_attention(c.q[:0], pre, 30, Q.KVPages(*c.suffix[:2], table=c.st[:0]), lens[:0], 20).shape == (0, 8, 64)


def test_attention_sizes_past_the_join(Q, gpu):
    """Rows of requests of up to n_q tokens are counted in 31 bits, with room for a workgroup's."""
    import ctypes
    fake = 0x10000   # sizes only: nothing is read
    pages = Q.q4k_kv_pages(fake, fake, 8, 4096, 1 << 20, 256, 128, 1 << 20, 256, 128, None, 0, 8)
    size = lambda requests: Q.lib().q4k_prefix_attn_workspace_bytes(ctypes.byref(Q.q4k_prefix_attn_args(  # noqa: E731
        0, 1, 1, 1, 8, 1.0, 4, requests, 1, fake, fake, 32, 32, ctypes.pointer(pages), 30000, None, None, 0, fake, 32, 32, None)))
    assert size(1 << 20) > 0 and size((1 << 31) - 1000) > 0
    assert size((1 << 31) - 1) == 0 and size((1 << 31) - 100) == 0

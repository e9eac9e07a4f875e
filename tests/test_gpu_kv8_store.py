"""q4k_kv8_store and q4k_kv8_load against the same steps in 64 bits: every byte, scale
and value, over types, head sizes, blocks, pages, new tokens and lengths."""
import pytest
import torch

import _step

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
I8, E4M3 = torch.int8, torch.float8_e4m3fn
KINDS = [I8, E4M3]


def as_bytes(values, dtype):
    return values.to(dtype) if dtype == I8 else values.float().to(dtype)


class Cache:
    """Pages of earlier tokens, some in every block, and its plain form beside it."""

    def __init__(self, gpu, kind, B, most, hk, D, page, block, seed=0, strided=False):
        self.g = g = torch.Generator(device=gpu).manual_seed(seed)
        self.gpu, self.kind, self.B, self.most, self.hk, self.D = gpu, kind, B, most, hk, D
        per = -(-most // page)
        n = B * per + 2
        self.t = []
        for _ in range(2):
            code = torch.randint(-127, 128, (n, page, hk, D), device=gpu, generator=g)
            x = code.to(I8) if kind == I8 else torch.sign(code) * _step.CODES.to(gpu)[code.abs().clamp(max=126)]
            x = x if kind == I8 else x.float().to(E4M3)
            if strided:  # [pages, heads, tokens, dim] with places between the rows
                room = torch.zeros(n, hk, page, D + 16, device=gpu, dtype=torch.uint8).view(kind)
                y = room[..., :D].transpose(1, 2)
                y.copy_(x)
                x = y
            self.t.append(x)
        self.t += [torch.rand(n, page // block, hk, device=gpu, generator=g) * 0.02 + 0.001 for _ in range(2)]
        self.table = torch.randperm(n, device=gpu, generator=g)[:B * per].view(B, per).int().contiguous()

    def pages(self, Q):
        return Q.KV8Pages(*self.t, table=self.table)

    def plain(self):
        return _step.Cache8(*self.t, self.table)

    def rows(self, n, dtype, mul=1.0):
        return [(torch.randn(n, self.hk, self.D, device=self.gpu, generator=self.g) * mul).to(dtype) for _ in range(2)]

    def check(self, want):
        for got, held, name in zip(self.t[:2], want.held, "kv"):
            bad = (got.cpu().float().double() != held) & ~(torch.isnan(got.cpu().float()) & torch.isnan(held))
            assert not bad.any(), f"{name}: {int(bad.sum())} bytes, first at {bad.nonzero()[0].tolist()}"
        for got, scale, name in zip(self.t[2:], want.scale, "kv"):
            assert torch.equal(got.cpu(), scale), f"{name}_scale"


def run(Q, c, n, spans, lens, dtype, ragged, mul=1.0, most_q=None):
    new = c.rows(n, dtype, mul)
    want = c.plain()
    want.store(new, spans, lens)
    start = torch.tensor([s[0] for s in spans] + [spans[-1][1]], dtype=torch.int32, device=c.gpu) if ragged else None
    l32 = torch.tensor(lens, dtype=torch.int32, device=c.gpu)
    n_q = most_q or max(b - a for a, b in spans)
    Q.kv8_store(c.pages(Q), *new, l32, c.most, n_q=n_q, q_start=start)
    c.check(want)
    return want, l32


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,n_q,most,hk,D,page,block", [
    (1, 1, 1, 1, 16, 1, 1), (3, 1, 40, 8, 128, 16, 16), (16, 1, 200, 2, 64, 64, 32), (2, 5, 100, 4, 80, 24, 12), (4, 3, 77, 2, 96, 20, 4),
    (2, 300, 700, 2, 128, 128, 64), (3, 33, 64, 1, 256, 32, 32), (1, 700, 900, 3, 48, 256, 256), (5, 2, 50, 8, 112, 48, 1), (2, 130, 300, 4, 64, 300, 100)])
def test_store(Q, gpu, kind, dtype, B, n_q, most, hk, D, page, block):
    for seed, mul in ((0, 1.0), (1, 8.0), (2, 0.1)):  # scales that change in some blocks, in all, in none
        c = Cache(gpu, kind, B, most, hk, D, page, block, seed=seed)
        lens = torch.randint(min(n_q, most), most + 1, (B,), generator=torch.Generator().manual_seed(seed)).tolist()
        lens[0] = most
        run(Q, c, B * n_q, [(r * n_q, r * n_q + n_q) for r in range(B)], lens, dtype, False, mul)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,block", [(128, 32), (80, 8), (256, 64)])
def test_store_rows_of_their_own_number(Q, gpu, kind, D, block):
    """Prompts and single tokens together; requests without new tokens; lengths shorter than the new tokens."""
    spans = [(2, 40), (40, 40), (40, 41), (41, 150), (150, 153)]
    for strided in (False, True):
        c = Cache(gpu, kind, 5, 256, 2, D, 64, block, seed=D, strided=strided)
        run(Q, c, 160, spans, [200, 60, 33, 60, 2], BF16, True)  # (109 new tokens, 60 places: the last 60)
        run(Q, c, 160, spans, [256, 0, 1, 109, 0], F32, True)
        run(Q, c, 160, spans, [100, 20, 64, 256, 65], F16, True, most_q=160)


@pytest.mark.parametrize("kind", KINDS)
def test_store_token_by_token(Q, gpu, kind):
    """A block filled one token a call: scales that grow now and then, earlier tokens rounded again."""
    c = Cache(gpu, kind, 3, 70, 2, 64, 32, 16, seed=4)
    grown = 0
    for step in range(1, 71):
        before = c.t[2].clone()
        run(Q, c, 3, [(0, 1), (1, 2), (2, 3)], [step, step, max(0, step - 20)], F32, False, mul=1.0 + step % 7 * 0.3)
        grown += int((c.t[2] != before).sum())
    assert grown > 70


@pytest.mark.parametrize("kind", KINDS)
def test_store_ties_zeros_and_values_that_are_not_finite(Q, gpu, kind):
    """Quotients at and beside the middles of neighbours; blocks of zeros, of smallest
    values, of infinities and NaN."""
    c = Cache(gpu, kind, 1, 64, 1, 256, 64, 16, seed=5)
    new = torch.zeros(64, 1, 256, device=gpu)
    if kind == I8:
        mids = torch.arange(-126, 126, device=gpu).float() + 0.5
    else:
        mids = ((_step.CODES[1:] + _step.CODES[:-1]) / 2).float().to(gpu)
        mids = torch.cat([mids, -mids])
    top = _step.TOP[kind]
    new[:16, 0, :mids.numel()] = mids
    new[0:16, 0, 255] = top                                     # scale 1: ties as they are
    s = torch.tensor(1.2345678, device=gpu)
    new[16:32, 0, :mids.numel()] = mids * s                     # rounded once, either side of the tie
    new[16:32, 0, 255] = top * s
    new[20] = new[20].nextafter(torch.full_like(new[20], float("inf")))
    new[21] = new[21].nextafter(torch.full_like(new[21], -float("inf")))
    new[32:48] = 0.0
    new[40, 0, :4] = torch.tensor([1e-45, -3e-45, 1e-40, 7e-39], device=gpu)
    new[48:, 0, :5] = torch.tensor([float("inf"), -float("inf"), float("nan"), 3.0, -0.0], device=gpu)
    want = c.plain()
    want.store((new, -new), [(0, 64)], [64])
    Q.kv8_store(c.pages(Q), new, -new, torch.tensor([64], dtype=torch.int32, device=gpu), 64, n_q=64)
    c.check(want)
    assert (c.t[2][int(c.table[0, 0]), 3] == torch.tensor(3.0).double().div(top).float().to(gpu)).all()


@pytest.mark.parametrize("kind", KINDS)
def test_store_pages_out_of_range_and_lengths_past_the_bound(Q, gpu, kind):
    c = Cache(gpu, kind, 3, 96, 2, 64, 16, 8, seed=6)
    c.table[0, 1] = -1
    c.table[1, 5] = 2 ** 31 - 1
    run(Q, c, 120, [(0, 40), (40, 80), (80, 120)], [40, 96, 50], F32, False)
    # lengths past max_len count as max_len, below 0 as none
    new = c.rows(3, F32)
    want = c.plain()
    want.store(new, [(0, 1), (1, 2), (2, 2)], [96, 96, 0])
    Q.kv8_store(c.pages(Q), *new, torch.tensor([1000, 2 ** 31 - 1, -7], dtype=torch.int32, device=gpu), 96)
    c.check(want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,n_q,most,hk,D,page,block", [(1, 1, 1, 1, 16, 1, 1), (3, 70, 64, 2, 80, 24, 12), (4, 5, 100, 8, 128, 32, 32), (2, 40, 40, 3, 256, 8, 4)])
def test_load(Q, gpu, kind, dtype, B, n_q, most, hk, D, page, block):
    c = Cache(gpu, kind, B, most, hk, D, page, block, seed=7)
    if B > 2:
        c.table[1, 0] = -3
    lens = [most] + [max(0, most - 7 * r - 1) for r in range(1, B)]
    l32 = torch.tensor(lens, dtype=torch.int32, device=gpu)
    for ragged in (False, True):
        spans = [(r * n_q, r * n_q + n_q) for r in range(B)]
        n, start = B * n_q, None
        if ragged:
            spans = [(a + 1, b - (r == B - 1)) for r, (a, b) in enumerate(spans)]
            spans = [(a, max(a, (spans[r + 1][0] if r + 1 < B else b))) for r, (a, b) in enumerate(spans)]
            start = torch.tensor([s[0] for s in spans] + [spans[-1][1]], dtype=torch.int32, device=gpu)
        out = [torch.full((n + 2, hk, D), 7.0, device=gpu, dtype=dtype)[:n] for _ in range(2)]
        whole = [torch.full((n, hk, D), 7.0, dtype=dtype) for _ in range(2)]
        Q.kv8_load(c.pages(Q), *out, l32, most, n_q=n_q, q_start=start)
        plain = c.plain()
        for r, (a, b) in enumerate(spans):
            k, v, ok = plain.values(r, lens[r])
            for w, x in zip(whole, (k, v)):
                x = torch.where(ok[:, None, None], x, 0.0).float().to(dtype)  # (the product of byte and scale is rounded to F32 first)
                m = min(lens[r], b - a)
                w[a:b] = 0
                if m:
                    w[b - m:b] = x[lens[r] - m:]
        for o, w in zip(out, whole):
            assert torch.equal(o.cpu(), w)
    # one of the two alone
    only = torch.empty(B * n_q, hk, D, device=gpu, dtype=dtype)
    both = [torch.empty_like(only) for _ in range(2)]
    Q.kv8_load(c.pages(Q), *both, l32, most, n_q=n_q)
    assert torch.equal(Q.kv8_load(c.pages(Q), None, only, l32, most, n_q=n_q)[1], both[1])
    assert torch.equal(Q.kv8_load(c.pages(Q), only, None, l32, most, n_q=n_q)[0], both[0])


def test_store_rows_of_a_fused_projection_and_pages_in_order(Q, gpu):
    """Rows with strides of their own at odd addresses; no table."""
    hk, D, n = 2, 64, 48
    for dtype in (F32, F16):
        qkv = torch.randn(n, 8 * D + 4 * D + 1, device=gpu).to(dtype)
        k, v = qkv[:, 513:513 + hk * D].view(n, hk, D), qkv[:, 641:641 + hk * D].view(n, hk, D)
        t = [torch.zeros(6, 16, hk, D, device=gpu, dtype=I8) for _ in range(2)] + [torch.zeros(6, 2, hk, device=gpu) for _ in range(2)]
        table = torch.arange(6, device=gpu).int().view(2, 3)
        want = _step.Cache8(*t, table)
        want.store((k, v), [(0, 24), (24, 48)], [24, 40])
        Q.kv8_store(Q.KV8Pages(*t), k, v, torch.tensor([24, 40], dtype=torch.int32, device=gpu), 48, n_q=24)
        assert torch.equal(t[0].cpu().double(), want.held[0]) and torch.equal(t[1].cpu().double(), want.held[1])
        assert torch.equal(t[2].cpu(), want.scale[0]) and torch.equal(t[3].cpu(), want.scale[1])


def test_store_and_load_in_a_graph_on_a_stream(Q, gpu):
    """A captured step follows new lengths and rows; every replay against eager calls."""
    c = Cache(gpu, E4M3, 4, 64, 2, 64, 16, 16, seed=9)
    eager = [t.clone() for t in c.t]
    pages, plain = c.pages(Q), Q.KV8Pages(*eager, table=c.table)
    new = c.rows(4, F32)
    lens = torch.tensor([1, 20, 33, 48], dtype=torch.int32, device=gpu)
    out, want = ([torch.empty(64, 2, 64, device=gpu) for _ in range(2)] for _ in range(2))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        Q.kv8_store(pages, *new, lens, 64)
        Q.kv8_load(pages, *out, lens, 64, n_q=16)
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        Q.kv8_store(plain, *new, lens, 64)
        Q.kv8_load(plain, *want, lens, 64, n_q=16)
        for a, b in zip(c.t, eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        lens += 1
        for x in new:
            x.mul_(1.3)

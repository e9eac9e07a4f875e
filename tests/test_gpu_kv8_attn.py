"""q4k_kv8_attn against 64 bits: types, head layouts and sizes, blocks and pages, lengths
from none to many, several queries a request, unseen bytes and scales of any
kind, rows that see nothing."""
import pytest
import torch

import _batch
import _batch_terms
import _step

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
I8, E4M3 = torch.int8, torch.float8_e4m3fn
TYPES = [(q, kv) for q in (F32, F16, BF16) for kv in (I8, E4M3)]


class Case:
    """A batch with its cache; bytes and scales that no query may see are the worst there are."""

    def __init__(self, gpu, B, nq, H, hk, D, most, page, block, qt=F32, kv=I8, seed=0, lens=None, spans=None, strided=False):
        self.g = g = torch.Generator(device=gpu).manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, device=gpu, generator=g)  # noqa: E731
        self.B, self.nq, self.D, self.most, self.kv, self.gpu = B, nq, D, most, kv, gpu
        self.spans = spans or [(r * nq, r * nq + nq) for r in range(B)]
        self.q = rnd(self.spans[-1][1], H, D).to(qt)
        self.q_start = torch.tensor([s[0] for s in self.spans] + [self.spans[-1][1]], dtype=torch.int32, device=gpu) if spans else None
        per = -(-most // page)
        n = B * per + 2
        self.lens = lens if lens is not None else torch.randint(0, most + 1, (B,), device=gpu, generator=g).tolist()
        self.table = torch.randperm(n, device=gpu, generator=g)[:B * per].view(B, per).int().contiguous()
        shape = (n, hk, page, D) if strided else (n, page, hk, D)
        self.t = [torch.full(shape, 0x7f, dtype=torch.uint8, device=gpu).view(kv) for _ in range(2)]
        if strided:
            self.t = [t.transpose(1, 2) for t in self.t]
        self.t += [torch.full((n, page // block, hk), float("nan"), device=gpu) for _ in range(2)]
        for r in range(B):
            for i in range(-(-self.lens[r] // page)):
                m = min(page, self.lens[r] - i * page)
                at = int(self.table[r, i])
                for t, s in zip(self.t[:2], self.t[2:]):
                    x = rnd(m, hk, D) * (40 if kv == I8 else 100)
                    t[at, :m] = x.round().clamp(-127, 127).to(I8) if kv == I8 else x.clamp(-448, 448).to(E4M3)
                    s[at, :-(-m // block)] = torch.rand(-(-m // block), hk, device=gpu, generator=g) * 0.04 / (1 if kv == I8 else 2.5) + 0.002
        self.scale = D ** -0.5

    def run(self, Q, **kw):
        lens = torch.tensor(self.lens, dtype=torch.int32, device=self.gpu)
        lse = torch.full(self.q.shape[:2], 7.0, device=self.gpu)
        out = Q.kv8_attention(self.q, Q.KV8Pages(*self.t, table=self.table), lens, self.most, n_q=self.nq, q_start=self.q_start, scale=self.scale,
                              lse=lse, **kw)
        return out, lse

    def check(self, Q, **kw):
        out, lse = self.run(Q, **kw)
        want, wl, tol, tl = _step.attention8(self.q, self.spans, _step.Cache8(*self.t, self.table), [min(max(x, 0), self.most) for x in self.lens], self.scale)
        if self.q.dtype == F16:  # results past F16's range are infinite in it
            want = torch.where(want.abs() >= 65520, torch.sign(want) * float("inf"), want)
        for x, y in ((out, want), (lse, wl)):
            assert torch.equal(torch.isnan(x).cpu(), torch.isnan(y))
        _batch.assert_close(out, want, tol, "out")
        _batch.assert_close(lse, wl, tl, "lse")
        return out, lse


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("B,nq,H,hk,D,most,page,block", [
    (1, 1, 1, 1, 16, 1, 1, 1), (1, 1, 4, 2, 64, 5, 16, 16), (3, 1, 32, 8, 128, 200, 64, 32), (5, 1, 28, 4, 80, 129, 48, 8), (4, 1, 8, 1, 256, 200, 32, 32),
    (2, 5, 24, 8, 64, 301, 24, 12), (7, 3, 6, 2, 96, 64, 20, 4), (17, 1, 16, 2, 128, 300, 100, 100), (3, 40, 4, 2, 48, 190, 64, 64), (1, 1, 8, 8, 128, 3001, 16, 16),
    (2, 1, 4, 1, 128, 2500, 36, 12), (33, 1, 64, 8, 128, 70, 32, 1), (2, 9, 4, 2, 256, 90, 12, 3), (2, 70, 3, 1, 112, 300, 128, 64)])
def test_kv8_attention_sizes(Q, gpu, qt, kv, B, nq, H, hk, D, most, page, block):
    Case(gpu, B, nq, H, hk, D, most, page, block, qt, kv, seed=B + D).check(Q)


@pytest.mark.parametrize("qt,kv", TYPES)
def test_kv8_attention_strides_and_pages_in_order(Q, gpu, qt, kv):
    c = Case(gpu, 3, 1, 8, 2, 64, 150, 32, 16, qt, kv, lens=[150, 33, 0], strided=True)
    want = c.check(Q)
    wide = torch.zeros(3, 8 * 64 + 65, device=gpu, dtype=qt)
    view = wide[:, 1:8 * 64 + 1].view(3, 8, 64)
    view.copy_(c.q)
    c.q, out = view, torch.full((8, 3, 64), 7.0, device=gpu, dtype=qt).transpose(0, 1)
    got = c.run(Q, out=out)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # the same cache with its pages in order
    at = c.table.long().flatten()
    lens = torch.tensor(c.lens, dtype=torch.int32, device=gpu)
    t = [x.contiguous().view(torch.uint8)[at].view(kv) if i < 2 else x[at] for i, x in enumerate(c.t)]
    assert torch.equal(Q.kv8_attention(c.q, Q.KV8Pages(*t), lens, c.most), want[0])


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("block", [16, 4])
def test_kv8_attention_lengths_around_a_step(Q, gpu, qt, kv, block):
    lens = [0, 1, 7, 8, 9, 31, 32, 33, 127, 128, 129, 255, 256, 257, 383, 385]
    Case(gpu, len(lens), 1, 8, 2, 128, 390, 48, block, qt, kv, lens=lens).check(Q)
    Case(gpu, len(lens), 3, 2, 2, 64, 390, 48, block, qt, kv, lens=lens).check(Q)


@pytest.mark.parametrize("qt,kv", TYPES)
def test_kv8_attention_queries_of_their_own_number(Q, gpu, qt, kv):
    spans = [(2, 5), (5, 5), (5, 6), (6, 43), (43, 44)]
    c = Case(gpu, 5, 40, 12, 4, 64, 90, 32, 16, qt, kv, lens=[10, 4, 0, 90, 33], spans=spans)
    c.q = torch.cat([c.q, c.q[:3]])  # tokens of no request in front and behind
    out = torch.full_like(c.q, 5.0)
    got, lse = c.run(Q, out=out)
    want, wl, tol, tl = _step.attention8(c.q, c.spans, _step.Cache8(*c.t, c.table), c.lens, c.scale)
    _batch.assert_close(got[2:44], want[2:44], tol[2:44], "out")
    _batch.assert_close(lse[2:44], wl[2:44], tl[2:44], "lse")
    assert (got[:2] == 5).all() and (got[44:] == 5).all() and (lse[:2] == 7).all() and (lse[44:] == 7).all()


@pytest.mark.parametrize("kv", [I8, E4M3])
@pytest.mark.parametrize("most", [40, 600])
def test_kv8_attention_rows_that_see_nothing(Q, gpu, kv, most):
    c = Case(gpu, 4, 3, 8, 2, 64, most, 20, 10, F32, kv, lens=[0, 1, 2, 40])
    out, lse = c.check(Q)
    assert not out[:3].any() and (lse[:3] == -float("inf")).all() and not out[3:5].any() and lse[5].isfinite().all()
    c.table.fill_(-1)
    out, lse = c.run(Q)
    assert not out.any() and (lse == -float("inf")).all()
    got = Q.kv8_attention(c.q, Q.KV8Pages(*c.t, table=c.table), torch.zeros(4, dtype=torch.int32, device=gpu), 0, n_q=3)
    assert not got.any()


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("block", [8, 4])
def test_kv8_attention_pages_out_of_range_and_lengths_past_the_bound(Q, gpu, qt, kv, block):
    c = Case(gpu, 3, 2, 8, 2, 128, 100, 8, block, qt, kv, lens=[100, 50, 33])
    c.table[0, 2], c.table[1, 0], c.table[0, 12] = -5, 2 ** 31 - 1, 10 ** 6
    want = c.check(Q)
    c.lens = [10 ** 9, 50, 33]
    got = c.run(Q)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    c.lens = [-7, 0, -2 ** 31]
    assert not c.run(Q)[0].any()


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("block", [16, 1])
@pytest.mark.parametrize("nq,most", [(4, 40), (40, 300)])
def test_kv8_attention_bytes_and_scales_behind_the_causal_bound(Q, gpu, qt, kv, block, nq, most):
    """What only the last query sees leaves the others alone."""
    c = Case(gpu, 2, nq, 4, 2, 64, most, 16, block, qt, kv, lens=[most, nq + 1])
    want = c.run(Q)
    for r, length in enumerate(c.lens):
        j = length - 1
        p, s = int(c.table[r, j // 16]), j % 16
        for t in c.t[:2]:
            t.view(torch.uint8)[p, s] = 0x7f
        if block == 1:
            c.t[2][p, s] = float("nan")
            c.t[3][p, s] = float("inf")
    got = c.run(Q)
    for r in range(2):
        lo, hi = r * nq, (r + 1) * nq - 1
        assert torch.equal(got[0][lo:hi], want[0][lo:hi]) and torch.equal(got[1][lo:hi], want[1][lo:hi])
        if kv == E4M3 or block == 1:
            assert torch.isnan(got[0][hi]).all()
    if kv == E4M3:  # a value alone, that several queries see
        c = Case(gpu, 2, nq, 4, 2, 64, most, 16, block, qt, kv, lens=[most, nq + 1])
        j = most - 2
        c.t[1].view(torch.uint8)[int(c.table[0, j // 16]), j % 16, 1, 5] = 0xff
        out, _ = c.run(Q)
        bad = torch.isnan(out)
        assert bad[nq - 2:nq, 2:, 5].all() and int(bad.sum()) == 4


@pytest.mark.parametrize("qt,kv", TYPES)
def test_kv8_attention_peaked_flat_and_large_scores(Q, gpu, qt, kv):
    c = Case(gpu, 6, 1, 8, 2, 128, 700, 64, 32, qt, kv, seed=3, lens=[700, 700, 690, 650, 700, 3])
    c.q[0] = 0                    # flat
    c.q[1] = c.q[1] * 30          # one position takes all
    c.t[2][c.table[2, 10].long()] *= 50   # keys late in the request
    c.t[3][c.table[3, 2].long()] *= 1e20  # values of very different scales
    c.t[3][c.table[4, 5].long()] *= 1e-30
    c.check(Q)
    c.scale = -c.scale
    c.check(Q)
    c.scale = 0.0
    c.check(Q)
    if qt == F32:
        for f in (1e-30, 1e30):
            c.q, c.scale = c.q * f, 0.05 / f
            c.check(Q)
            c.q = c.q / f


def test_kv8_attention_scores_keep_f32(Q, gpu):
    """One key and one dimension a query: the log-sum-exp is the score, at a bound
    that one F16 term would miss (its 2^-12 is 200 times it)."""
    U = _batch_terms.U
    g = torch.Generator(device=gpu).manual_seed(1)
    for kv in (I8, E4M3):
        for B, H, hk, D in ((3, 8, 2, 128), (5, 4, 4, 256), (9, 3, 1, 80)):
            at = torch.randint(0, D, (B, H), device=gpu, generator=g)
            value = _batch_terms.full((B, H), g, gpu, 3, 6)
            q = torch.zeros(B, H, D, device=gpu).scatter_(2, at[:, :, None], value[:, :, None])
            k = torch.randint(1, 120, (B, 16, hk, D), device=gpu, generator=g).float().to(kv)
            s = [torch.rand(B, 1, hk, device=gpu, generator=g) * 0.01 + 0.005 for _ in range(2)]
            lse = torch.empty(B, H, device=gpu)
            Q.kv8_attention(q, Q.KV8Pages(k, k, *s), torch.ones(B, dtype=torch.int32, device=gpu), 16, scale=1.0, lse=lse)
            kd = (k[:, 0].float().double() * s[0].double().transpose(1, 2)).repeat_interleave(H // hk, 1)
            want = value.double() * kd.gather(2, at[:, :, None])[:, :, 0]
            # two F16 terms 2^-22, then the sum, scale, factor, reference and difference: below 10 units
            _batch.assert_close(lse, want.cpu(), (10 * U * want.abs() + 2.0 ** -18).cpu(), "score")


def test_kv8_attention_probabilities_keep_f32(Q, gpu):
    """One position a dimension of the values: a result is a single probability times
    a value, at the bound of _batch_terms' probabilities and a unit for the scale."""
    U = _batch_terms.U
    g = torch.Generator(device=gpu).manual_seed(2)
    for kv in (I8, E4M3):
        for B, H, hk, D, n in ((3, 8, 2, 128, 33), (2, 34, 1, 64, 64), (5, 4, 2, 256, 5)):
            at = torch.randint(0, D, (B, H), device=gpu, generator=g)
            value = _batch_terms.full((B, H), g, gpu, -2, -1)
            q = torch.zeros(B, H, D, device=gpu).scatter_(2, at[:, :, None], value[:, :, None])
            k = torch.randint(-120, 121, (B, 64, hk, D), device=gpu, generator=g).float().to(kv)
            v = torch.zeros(B, 64, hk, D, device=gpu)
            d = torch.arange(D, device=gpu)
            v[:, d % n, :, d] = torch.randint(1, 120, (D, B, hk), device=gpu, generator=g).float()
            v = v.to(kv)
            s = [torch.rand(B, 4, hk, device=gpu, generator=g) * 0.01 + 0.005 for _ in range(2)]
            got = Q.kv8_attention(q, Q.KV8Pages(k, v, *s), torch.full((B,), n, dtype=torch.int32, device=gpu), 64, scale=1.0)
            kd, vd = ((x.float().double() * y.double().repeat_interleave(16, 1)[..., None])[:, :n].repeat_interleave(H // hk, 2) for x, y in zip((k, v), s))
            score = value.double()[:, :, None] * kd.permute(0, 2, 3, 1).gather(2, at[:, :, None, None].expand(B, H, 1, n))[:, :, 0]
            p = torch.softmax(score, 2)                                          # [B, H, n]
            want = p[:, :, d % n] * vd[:, d % n, :, d].permute(1, 2, 0)
            _batch.assert_close(got, want.cpu(), (61 * U * want.abs() + 1e-30).cpu(), f"probability of {n}")


def test_kv8_attention_workspaces_streams_and_graphs(Q, gpu):
    c = Case(gpu, 5, 1, 16, 4, 128, 2000, 64, 32, BF16, E4M3, lens=[2000, 900, 1, 0, 1999])
    lens = torch.tensor(c.lens, dtype=torch.int32, device=gpu)
    pages = Q.KV8Pages(*c.t, table=c.table)
    ws = Q.kv8_attention_workspace(c.q, pages, lens, c.most)
    assert ws.numel() > 16
    ws.fill_(255)
    want, lse = c.check(Q)
    got = c.run(Q, workspace=ws)
    assert torch.equal(got[0], want) and torch.equal(got[1], lse)
    with pytest.raises(Q.Q4KError):
        c.run(Q, workspace=ws[:-16])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = Q.kv8_attention(c.q, pages, lens, c.most, scale=c.scale, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    # two captured graphs with a workspace each, replayed by turns, follow the lengths
    outs, graphs, keep = [], [], []
    for i in range(2):
        outs.append(torch.empty_like(c.q))
        w = torch.empty_like(ws)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            Q.kv8_attention(c.q, pages, lens, c.most, scale=c.scale, out=outs[i], workspace=w)
        keep.append(w)
    for step in range(4):
        lens.copy_(torch.tensor([2000 - step * 300, 900, step, 0, 1999 - 500 * step]))
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        c.lens = lens.tolist()
        want = c.run(Q)[0].view(torch.int16)  # (bits: a length past what was filled reads NaN)
        assert torch.equal(outs[0].view(torch.int16), want) and torch.equal(outs[1].view(torch.int16), want)
        c.q.mul_(0.9)


def test_kv8_attention_a_step_with_rope_and_store(Q, gpu):
    """As a server runs them: norms and rotation, the new keys and values into the cache,
    attention; prompts of several lengths first, then tokens one by one."""
    B, H, hk, D, page, block, most = 3, 8, 2, 64, 32, 16, 96
    g = torch.Generator(device=gpu).manual_seed(8)
    for kv in (I8, E4M3):
        t = [torch.zeros(B * 3, page, hk, D, device=gpu, dtype=torch.uint8).view(kv) for _ in range(2)]
        t += [torch.zeros(B * 3, page // block, hk, device=gpu) for _ in range(2)]
        table = torch.randperm(B * 3, device=gpu, generator=g).view(B, 3).int()
        pages, plain = Q.KV8Pages(*t, table=table), _step.Cache8(*t, table)
        w = 1 + 0.2 * torch.randn(D, device=gpu, generator=g)
        rope = Q.Rope(D, mode="neox", q_norm=w, k_norm=w)
        lens = torch.zeros(B, dtype=torch.int32, device=gpu)
        for step in range(6):
            n = [20, 1, 47] if step == 0 else [1, 1, 1]
            start = torch.tensor([0, n[0], n[0] + n[1], sum(n)], dtype=torch.int32, device=gpu)
            spans = list(zip(start.tolist(), start.tolist()[1:]))
            lens += start.diff()
            pos = torch.cat([torch.arange(int(lens[r]) - n[r], int(lens[r]), device=gpu) for r in range(B)]).int()
            q, k, v = (torch.randn(sum(n), h, D, device=gpu, generator=g) for h in (H, hk, hk))
            q, k = Q.rope(rope, q, k, pos, q_out=q, k_out=k)
            Q.kv8_store(pages, k, v, lens, most, n_q=max(n), q_start=start)
            plain.store((k, v), spans, lens.tolist())
            assert torch.equal(t[0].cpu().float().double(), plain.held[0]) and torch.equal(t[3].cpu(), plain.scale[1])
            out = Q.kv8_attention(q, pages, lens, most, n_q=max(n), q_start=start)
            want, _, tol, _ = _step.attention8(q, spans, plain, lens.tolist(), D ** -0.5)
            _batch.assert_close(out, want, tol, f"step {step}")


@pytest.mark.parametrize("qt,kv", TYPES)
@pytest.mark.parametrize("B,nq,H,hk,D,most,page,block", [
    (40, 1, 8, 8, 64, 1300, 32, 16), (300, 1, 8, 8, 32, 300, 20, 4), (600, 2, 4, 4, 16, 290, 16, 16), (9, 1, 16, 8, 256, 1900, 64, 64), (20, 20, 16, 4, 128, 1200, 48, 12)])
def test_kv8_attention_dealt_out(Q, gpu, qt, kv, B, nq, H, hk, D, most, page, block):
    """Enough positions for every workgroup to take steps of several requests and heads,
    of more requests than a workgroup counts at once; requests of none and of one."""
    lens = [(i * 7919 + 13) % (most + 1) for i in range(B)]
    lens[0], lens[1], lens[B - 1], lens[B // 2] = 0, 1, most, 0
    Case(gpu, B, nq, H, hk, D, most, page, block, qt, kv, seed=B + D, lens=lens).check(Q)


@pytest.mark.parametrize("lens", [[0] * 64, [0] * 63 + [4000], [4000] + [1] * 63, [128] * 64, [129] * 64])
def test_kv8_attention_dealt_out_of_one_request(Q, gpu, lens):
    """Bounds far past the lengths: all of the work in one request, or in none."""
    case = Case(gpu, 64, 1, 8, 2, 64, 4000, 64, 32, BF16, E4M3, seed=3, lens=lens)
    out, _ = case.check(Q)
    assert torch.equal(out, case.run(Q)[0])


def test_kv8_attention_dealt_out_ragged_in_a_graph(Q, gpu):
    """Requests of their own numbers of tokens, with rows of none before, between and behind them,
    replayed with other lengths."""
    B, most = 48, 1500
    spans, at = [], 3
    for i in range(B):
        spans.append((at, at + (0, 1, 5, 2)[i % 4]))
        at = spans[-1][1]
    case = Case(gpu, B, 5, 16, 8, 64, most, 32, 8, F16, I8, seed=5, spans=spans, lens=[0] * B)
    pages = Q.KV8Pages(*case.t, table=case.table)
    q = torch.cat([case.q, case.q[:4]])
    lens = torch.tensor([0] * B, dtype=torch.int32, device=gpu)
    full = torch.randint(1, most, (B,), generator=torch.Generator().manual_seed(1)).int()
    for t, s in zip(case.t[:2], case.t[2:]):
        t.view(torch.uint8).copy_(torch.randint(0, 120, t.shape, device=gpu, generator=case.g).to(torch.uint8))
        s.copy_(torch.rand(s.shape, device=gpu, generator=case.g) * 0.01)
    ws = Q.kv8_attention_workspace(q, pages, lens, most, n_q=5, q_start=case.q_start)
    out, lse = torch.full_like(q, 3.0), torch.full(q.shape[:2], 4.0, device=gpu)
    call = dict(n_q=5, q_start=case.q_start, scale=case.scale, out=out, lse=lse, workspace=ws)
    Q.kv8_attention(q, pages, lens, most, **call)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        Q.kv8_attention(q, pages, lens, most, **call)
    for i in range(4):
        lens.copy_((full * (i + 1) // 4).to(gpu))
        graph.replay()
        torch.cuda.synchronize()
        eager = Q.kv8_attention(q, pages, lens, most, **dict(call, out=torch.full_like(q, 3.0), lse=None, workspace=None))
        assert torch.equal(out, eager)
        n = case.q.shape[0]
        assert (out[:3] == 3).all() and (out[n:] == 3).all() and (lse[:3] == 4).all() and (lse[n:] == 4).all()
        want, wl, tol, tl = _step.attention8(case.q, spans, _step.Cache8(*case.t, case.table), lens.tolist(), case.scale)
        _batch.assert_close(out[3:n], want[3:], tol[3:], "out")
        _batch.assert_close(lse[3:n], wl[3:], tl[3:], "lse")


def test_kv8_attention_more_steps_than_are_counted(Q, gpu):
    """(host checks alone: no workspace is named for what a call would refuse)"""
    k = torch.zeros(64, device=gpu)
    lens = torch.zeros(1, dtype=torch.int32, device=gpu)
    args = Q.q4k_kv8_attn_args()
    pages = Q.q4k_kv8_pages(Q.TYPE_I8, 300, 16, 1 << 30, k.data_ptr(), k.data_ptr(), 1, 1 << 30, 16, 16, 16, 16, 16, 16, k.data_ptr(), k.data_ptr(), 4, 4, 4, None, 0, 1)
    import ctypes
    for heads, some in ((300, False), (100, True)):
        pages.n_head_kv = heads
        args = Q.q4k_kv8_attn_args(ctypes.pointer(pages), Q.GGML_TYPE_F32, heads, 1.0, 1, 1, 1, None, lens.data_ptr(), 1 << 30, k.data_ptr(), 64, 64, k.data_ptr(), 64, 64, None)
        assert (Q.lib().q4k_kv8_attn_workspace_bytes(ctypes.byref(args)) > 0) == some

"""q4k_sample against 64 bits: sizes, every combination of rules, ties, flat and peaked
rows, masked rows, values that are not finite, borders of the sums."""
import itertools

import pytest
import torch

import _step

pytestmark = pytest.mark.gpu


def check(Q, x, u, t=None, k=None, p=None, m=None, lost=0, **kw):
    """Every row's token and log-probability; rows whose choice hangs on less than
    2^-36 of a sum are left out, at most `lost` of them."""
    n = x.shape[0]
    dev = x.device
    f = lambda v, d: None if v is None else torch.tensor(v, dtype=d, device=dev)  # noqa: E731
    lp = torch.full((n,), 7.0, device=dev)
    tokens, got = Q.sample(x, f(u, torch.float32), f(t, torch.float32), f(k, torch.int32), f(p, torch.float32), f(m, torch.float32), logprob=lp, **kw)
    assert got is lp and tokens.dtype == torch.int32
    as32 = lambda v, d: d if v is None else float(torch.tensor(v, dtype=torch.float32))  # noqa: E731
    left = 0
    for i in range(n):
        at = lambda v: None if v is None else v[i]  # noqa: E731
        want, w, margin = _step.sample(x[i], None if u is None else as32(u[i], 0.0), as32(at(t), 1.0), 0 if k is None else k[i], as32(at(p), 1.0), as32(at(m), 0.0))
        if margin < 2.0 ** -36:
            left += 1
            continue
        assert int(tokens[i]) == want, (i, int(tokens[i]), want, at(t), at(k), at(p), at(m), at(u))
        # a unit of F32, and what 64-bit sums of 2^18 terms leave
        assert float(lp[i]) == w or abs(float(lp[i]) - w) <= 2.0 ** -24 * abs(w) + 1e-10, (i, float(lp[i]), w)
    assert left <= lost
    return tokens, lp


def logits(gpu, n, V, seed, spread=2.5):
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.randn(n, V, device=gpu, generator=g) * spread
    x[:, ::17] = -float("inf")
    return x, torch.rand(n, device=gpu, generator=g).tolist()


@pytest.mark.parametrize("V", [1, 2, 5, 64, 255, 256, 257, 1000, 4097, 32768, 50257, 128256, 151936])
def test_sample_sizes_and_rules(Q, gpu, V):
    rules = list(itertools.product([1.0, 0.6], [0, 1, 7, 50], [1.0, 0.9, 0.3], [0.0, 0.05]))
    x, u = logits(gpu, len(rules), V, V)
    if V == 1:
        x.fill_(0.5)
    t, k, p, m = (list(c) for c in zip(*rules))
    check(Q, x, u, t, k, p, m)
    check(Q, x, u)
    check(Q, x, None, t, k, p, m)


@pytest.mark.parametrize("spread", [0.0, 1e-6, 0.01, 0.3, 10.0, 300.0])
def test_sample_flat_and_peaked_rows(Q, gpu, spread):
    """Thousands of logits in one bin, and few in all of them; large top-k."""
    for V in (3000, 40000):
        rules = [(0, 1.0), (1500, 1.0), (0, 0.5), (2000, 0.7), (2999, 0.99), (1024, 0.01), (20, 0.3), (1, 1.0)]
        x, u = logits(gpu, len(rules), V, V, spread)
        x += 3
        check(Q, x, u, [1.0] * len(rules), *(list(c) for c in zip(*rules)))
        check(Q, x, u, [0.05, 20.0] * 4, *(list(c) for c in zip(*rules)), [0.1, 0.0, 0.9, 1.0] * 2)


def test_sample_ties_go_to_lower_tokens(Q, gpu):
    """Equal logits, more of them than a list holds too, with sums that are whole numbers."""
    for V, steps in ((16, 1), (5000, 1), (5000, 3), (40000, 2), (3000, 2900)):
        x = (torch.arange(V, device=gpu) * 7919 % steps).float().repeat(6, 1) * -40.0 + 2.0   # groups of equal ones, 2^-57 apart
        n = int((x[0] == 2).sum())
        for half in (0.25, 0.5, 0.75):
            u = [0.0, 0.25, 0.5, 0.75, 0.9999, 0.5]
            tokens, lp = Q.sample(x, torch.tensor(u, device=gpu), top_k=torch.tensor([max(1, int(n * half))] * 6, dtype=torch.int32, device=gpu),
                                  logprob=torch.empty(6, device=gpu))
            at = (x[0] == 2).nonzero()[:, 0][:max(1, int(n * half))]
            assert tokens.tolist() == [int(at[int(v * at.numel())]) for v in torch.tensor(u).tolist()]
            assert torch.allclose(lp, torch.full_like(lp, -1.0) * torch.log(torch.tensor(float(at.numel()))).to(gpu), rtol=2.0 ** -23, atol=0)
            if steps == 1:
                # top-p of n equal tokens: those before which less than p n lies
                tokens, _ = Q.sample(x, torch.tensor(u, device=gpu), top_p=torch.full((6,), half, device=gpu))
                at = (x[0] == 2).nonzero()[:, 0][:-int(-n * half // 1)]
                assert tokens.tolist() == [int(at[int(v * at.numel())]) for v in torch.tensor(u).tolist()]
    x = torch.tensor([[0.0, -0.0, 0.0, -1.0]], device=gpu).repeat(3, 1)
    one = torch.ones(3, dtype=torch.int32, device=gpu)
    assert Q.sample(x, torch.tensor([0.0, 0.5, 0.99], device=gpu), top_k=one * 2)[0].tolist() == [0, 1, 1]
    assert Q.sample(x)[0].tolist() == [0, 0, 0]


def test_sample_rows_that_leave_nothing_or_one(Q, gpu):
    inf, nan = float("inf"), float("nan")
    V = 700
    x = torch.full((8, V), -inf, device=gpu)
    x[1, 300] = -5.0
    x[2] = nan
    x[3, 699] = inf
    x[4, 3], x[4, 600], x[4, 5] = inf, inf, 100.0
    x[5] = torch.randn(V, device=gpu)
    x[5, ::3] = nan
    x[6, 10], x[6, 20] = 3e38, -3e38
    x[7, 4] = -3.4e38
    for kw in (dict(), dict(k=[2] * 8), dict(p=[0.9] * 8), dict(m=[0.5] * 8), dict(k=[1] * 8, p=[0.1] * 8, m=[1.0] * 8), dict(t=[0.0] * 8), dict(t=[1e-30] * 8),
               dict(t=[1e30] * 8, p=[0.6] * 8)):
        tokens, lp = check(Q, x, [0.7] * 8, **kw)
        assert tokens[[0, 2]].tolist() == [-1, -1] and (lp[[0, 2]] == -inf).all() and tokens[[1, 3, 7]].tolist() == [300, 699, 4]
    assert Q.sample(x)[0].tolist()[:5] == [-1, 300, -1, 699, 3]
    empty = torch.empty(3, 0, device=gpu)
    assert Q.sample(empty, torch.rand(3, device=gpu))[0].tolist() == [-1, -1, -1]
    assert Q.sample(torch.empty(0, 50, device=gpu), torch.empty(0, device=gpu))[0].shape == (0,)


def test_sample_rules_out_of_range(Q, gpu):
    nan, inf = float("nan"), float("inf")
    x, _ = logits(gpu, 1, 500, 3)
    x = x.repeat(12, 1)
    u = [0.0, 1.0, 2.0, -1.0, nan, 0.3, 0.3, 0.3, 0.3, 0.3, 0.3, 0.3]
    t = [1.0] * 6 + [-1.0, nan, inf, 1.0, 1.0, 1.0]
    k = [0, 0, 0, 0, 0, -5, 3, 3, 3, 10 ** 9, 0, 0]
    p = [1.0, 1.0, 1.0, 1.0, 1.0, nan, 0.5, 0.5, 0.5, 5.0, -1.0, 0.0]
    m = [0.0] * 5 + [nan, -1.0, 7.0, 0.0, 0.0, 0.0, 7.0]
    check(Q, x, u, t, k, p, m)


def test_sample_follows_the_distribution(Q, gpu):
    """Uniform numbers on a fine grid draw each token as often as its share says, to
    one draw at either end of its stretch."""
    n = 4000
    x = torch.tensor([0.3, -1.0, 2.0, 1.5, -0.2, 0.9], device=gpu)
    u = (torch.arange(n, device=gpu) + 0.5) / n
    for k, p, kept in ((0, 1.0, [0, 1, 2, 3, 4, 5]), (3, 1.0, [2, 3, 5]), (0, 0.6, [2, 3])):
        tokens, _ = Q.sample(x.repeat(n, 1), u, temperature=torch.full((n,), 0.8, device=gpu), top_k=torch.full((n,), k, dtype=torch.int32, device=gpu),
                             top_p=torch.full((n,), p, device=gpu))
        share = torch.softmax(x[kept].double().cpu() / float(torch.tensor(0.8)), 0)
        have = torch.bincount(tokens.long().cpu(), minlength=6).double()
        assert have.sum() == have[kept].sum() and (have[kept] - share * n).abs().max() <= 1
        assert (tokens.diff() >= 0).all()


def test_sample_strides_streams_and_graphs(Q, gpu):
    x, u = logits(gpu, 9, 5003, 4)
    t, k, p, m = [0.7] * 9, [0, 40, 0, 9, 300, 0, 1, 2, 3], [0.9, 1.0, 0.5] * 3, [0.0, 0.02, 0.0] * 3
    want, lp = check(Q, x, u, t, k, p, m)
    for off in (1, 2, 3):
        wide = torch.full((9, 5003 + 7), float("inf"), device=gpu)
        view = wide[:, off:off + 5003]
        view.copy_(x)
        got = check(Q, view, u, t, k, p, m)
        assert torch.equal(got[0], want) and torch.equal(got[1], lp)
    dev = [torch.tensor(v, device=gpu, dtype=d) for v, d in ((u, torch.float32), (t, torch.float32), (k, torch.int32), (p, torch.float32), (m, torch.float32))]
    ws = Q.sample_workspace(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = Q.sample(x, *dev, stream=s)[0]
    s.synchronize()
    assert torch.equal(got, want)
    out, olp = torch.empty_like(want), torch.empty_like(lp)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        Q.sample(x, *dev, out=out, logprob=olp, workspace=ws)
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        e = torch.empty_like(lp)
        assert torch.equal(out, Q.sample(x, *dev, logprob=e)[0]) and torch.equal(olp, e)
        x.mul_(0.8)
        dev[0].copy_(torch.rand(9, device=gpu))
        dev[1].fill_(0.0 if i == 1 else 0.9)


def test_sample_many_rows_after_the_rules_of_the_logits(Q, gpu):
    """As a server runs them: penalties and masks in place, then the tokens."""
    n, V = 300, 2000
    x, u = logits(gpu, n, V, 6)
    mask = torch.randint(-2 ** 31, 2 ** 31, (n, -(-V // 32)), device=gpu, generator=torch.Generator(device=gpu).manual_seed(6)).int()
    mask[7] = 0
    Q.logits_adjust(x, mask=mask, out=x)
    tokens, _ = check(Q, x, u, [0.8] * n, [0, 50, 5] * 100, [0.95, 1.0] * 150, [0.0, 0.0, 0.01] * 100)
    ok = tokens.long().clamp(min=0)
    assert int(tokens[7]) == -1
    bit = (mask.gather(1, (ok // 32)[:, None])[:, 0] >> (ok % 32)) & 1
    assert ((bit == 1) | (tokens < 0)).all()


@pytest.mark.parametrize("V,spread", [(128256, 2.0), (151936, 0.2), (262144, 4.0), (262145, 2.0), (300001, 0.05)])
def test_sample_large_vocabularies(Q, gpu, V, spread):
    """Cuts that keep few tokens and many, two of them past what a list holds, bounds
    alone; rows of more tokens than a scan numbers."""
    rules = [(1.0, 5000, 1.0, 0.0), (1.0, 5000, 0.9, 0.0), (0.8, 0, 0.99, 0.0), (1.2, 0, 0.9, 0.02), (1.0, 0, 1.0, 0.3), (1.0, 0, 1.0, 1e-4), (1.0, 0, 1.0, 1.0),
             (0.7, 40, 0.95, 0.05), (0.7, 200, 0.8, 0.0), (1.0, 1024, 1.0, 0.0), (1.0, 1025, 0.5, 0.0), (0.05, 0, 0.5, 0.0), (50.0, 3, 0.5, 0.1), (1.0, 0, 1.0, 0.0)]
    x, u = logits(gpu, len(rules), V, V, spread)
    t, k, p, m = (list(c) for c in zip(*rules))
    check(Q, x, u, t, k, p, m)
    # what a mask leaves, by the lowest value instead of infinities: a range of 2^128
    x[:, torch.arange(V, device=gpu) % 50 != 3] = torch.finfo(torch.float32).min
    check(Q, x, u, t, k, p, m)


def test_sample_logits_out_of_a_scans_reach(Q, gpu):
    """a l past what the bins number, of the largest logit, of parts alone and of all."""
    V = 60000
    rules = [(1.0, 0, 1.0, 0.0), (1.0, 50, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.1), (1.0, 2000, 1.0, 0.0), (1.0, 1, 1.0, 0.0)]
    t, k, p, m = (list(c) for c in zip(*rules))
    for seed, f in enumerate((lambda x: x + 4000.0, lambda x: x - 1e5, lambda x: x * 1e4, lambda x: torch.where(x < 0, x - 1e6, x), lambda x: x * 1e-30)):
        x, u = logits(gpu, len(rules), V, seed, 1.0)
        check(Q, f(x), u, t, k, p, m)
        check(Q, f(x), u, [1e-4] * len(rules), k, p, m)


def test_sample_calls_at_once_and_again(Q, gpu):
    """Equal bits whatever runs beside a call, each with a workspace of its own."""
    n, V = 40, 50257
    x, u = logits(gpu, n, V, 12)
    rules = dict(temperature=torch.full((n,), 0.9, device=gpu), top_k=torch.tensor([0, 50] * 20, dtype=torch.int32, device=gpu),
                 top_p=torch.tensor([0.9] * 30 + [1.0] * 10, device=gpu), min_p=torch.tensor([0.0] * 35 + [0.01] * 5, device=gpu))
    u = torch.tensor(u, device=gpu)
    want, lp = Q.sample(x, u, logprob=torch.empty(n, device=gpu), **rules)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    spaces = [Q.sample_workspace(x) for _ in streams]
    got = []
    for i in range(12):
        s = streams[i % 3]
        with torch.cuda.stream(s):
            got.append(Q.sample(x, u, logprob=torch.empty(n, device=gpu), workspace=spaces[i % 3], **rules))
    torch.cuda.synchronize()
    for tokens, l in got:
        assert torch.equal(tokens, want) and torch.equal(l, lp)


def test_sample_more_rows_than_workgroups_at_once(Q, gpu):
    n, V = 600, 20000
    x, u = logits(gpu, n, V, 14, 1.5)
    check(Q, x, u, [0.9, 1.0, 0.0] * 200, [0, 40, 3000, 0, 0, 0] * 100, [0.95, 1.0, 0.9, 0.5, 1.0, 1.0] * 100, [0.0, 0.0, 0.0, 0.0, 0.2, 0.0] * 100)

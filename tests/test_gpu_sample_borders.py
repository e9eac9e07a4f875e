"""q4k_sample where tokens weigh next to nothing: weights at the end of what is numbered,
sums of small weights beside large ones, random numbers of 0 and near it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1.0, 0.37])
@pytest.mark.parametrize("chunks", [2, 5])
def test_sample_of_a_first_chunk_at_the_end_of_the_bins(Q, gpu, T, chunks):
    """A first chunk whose largest logit weighs about 2^-63 and 2^-64 of the row's, and a random
    number of 0: a token of the first chunk, or the first one of the next, never none."""
    steps = torch.arange(-200, 201, device=gpu) * 0.001
    for top in (0.0, 5.3, -2.25):
        for low in (-43.7, -44.36):
            for rest in (-float("inf"), None):
                x = torch.full((steps.numel(), chunks * 256), -float("inf"), device=gpu)
                x[:, 256:] = top
                x[:, 0] = top + (low + steps) * T
                if rest is None:  # all of the chunk's tokens alike
                    x[:, :256] = x[:, :1]
                n = x.shape[0]
                t = torch.full((n,), T, device=gpu)
                for u in (0.0, -1.0, float("nan")):
                    lp = torch.full((n,), 7.0, device=gpu)
                    got, _ = Q.sample(x, torch.full((n,), u, device=gpu), temperature=t, logprob=lp)
                    assert ((got == 0) | (got == 256)).all(), got.unique()
                    # what weighs 2^-63 and more is drawn, what weighs less than half of that is not
                    w = (x[:, 0].double() - top) / float(t[0]) / math.log(2)
                    assert (got[w >= -63] == 0).all() and (got[w < -64.1] == 256).all()
                    total = (chunks - 1) * 256
                    want = torch.where(got == 0, w * math.log(2), 0.0) - math.log(total)
                    assert ((lp - want).abs() <= 2.0 ** -24 * want.abs() + 1e-10).all()


def drawn(x, t, u, kept):
    """(token, log-probability, margin) of a row for each random number of u (all F32 values, in 64 bits):
    weights of the kept tokens in their order, sums without a rounding of their own; the margin is how far from
    u times the whole sum, in parts of it, the nearest token's sum lies."""
    w = [math.exp((float(x[i]) - float(x.max())) / t) for i in kept]
    upto, total = [], math.fsum(w)
    for i in range(len(w)):
        upto.append(math.fsum(w[:i + 1]))
    out = []
    for v in u:
        border = v * total
        n = next(i for i, s in enumerate(upto) if s > border)
        margin = min((abs(s - border) / border for s in upto[:-1]), default=1.0) if border else 1.0
        out.append((kept[n], math.log(w[n] / total), margin))
    return out


def check(Q, gpu, x, t, u, kept, k=0, p=1.0, m=0.0):
    """Each random number of u on the row x, but for those nearer than 2^-38 of it to a border."""
    n = len(u)
    t, p, m = (float(torch.tensor(v, dtype=torch.float32)) for v in (t, p, m))
    u = torch.tensor(u, dtype=torch.float32).tolist()
    full = lambda v, d=torch.float32: torch.full((n,), v, dtype=d, device=gpu)  # noqa: E731
    lp = full(7.0)
    got, _ = Q.sample(x.to(gpu).repeat(n, 1), torch.tensor(u, device=gpu), temperature=full(t), top_k=full(k, torch.int32), top_p=full(p), min_p=full(m), logprob=lp)
    tested = 0
    for i, (token, w, margin) in enumerate(drawn(x, t, u, kept)):
        if margin < 2.0 ** -38:
            continue
        tested += 1
        assert int(got[i]) == token, (i, u[i], int(got[i]), token, margin)
        assert abs(float(lp[i]) - w) <= 2.0 ** -24 * abs(w) + 1e-10, (i, float(lp[i]), w)
    assert tested * 2 > n


def test_sample_draws_what_a_cut_keeps_however_little_it_weighs(Q, gpu):
    x = torch.tensor([-4.0, 0.0])
    check(Q, gpu, x, 0.1, [0.0, 1e-30, 0.5], [0, 1], k=2)
    check(Q, gpu, torch.cat([x, torch.full((300,), -8.0)]), 0.1, [0.0, 1e-30, 1e-18, 0.5], [0, 1], k=2)
    check(Q, gpu, torch.cat([x, x - 0.01]), 0.1, [0.0, 0.5, 0.99], [0, 1, 3], k=3)


@pytest.mark.parametrize("n", [3, 200, 256, 257, 600, 1024])
@pytest.mark.parametrize("deep", [10, 30, 45, 60])
def test_sample_small_weights_of_a_list_add_up(Q, gpu, n, deep):
    """n - 1 tokens of about 2^-deep each, and behind them one of 1, kept by top-k, by top-k and top-p (all of
    them: the part is 1 - 2^-24 of a sum that lacks less), or by min-p too: random numbers that fall among the small ones."""
    g = torch.Generator().manual_seed(n + deep)
    for V in (2048, 40000):
        x = torch.full((V,), -200.0)
        at = torch.sort(torch.randperm(1024, generator=g)[:n - 1])[0]
        x[at] = -(deep - 1.5 * torch.rand(n - 1, generator=g)) * math.log(2)
        last = int(torch.randint(1280, V, (1,), generator=g))
        x[last] = 0.0
        kept = [*at.tolist(), last]
        small = math.fsum(math.exp(float(x[i])) for i in at.tolist())
        u = [0.0] + [small * v / (1 + small) for v in (1e-6, 1e-3, 0.1, 0.25, 0.5, 0.77, 0.9, 0.999, 1.3, 100.0)] + [0.7]
        u = [v for v in u if v < 1]
        check(Q, gpu, x, 1.0, u, kept, k=n)
        if n > 3:
            check(Q, gpu, x, 1.0, u, kept, k=n, m=2.0 ** -62)
            if deep > 30:
                check(Q, gpu, x, 1.0, u, [last], k=n, p=1 - 2.0 ** -24)


@pytest.mark.parametrize("rules", [dict(), dict(k=300), dict(m=2.0 ** -62), dict(k=40)])
@pytest.mark.parametrize("V,seed", [(256, 0), (3000, 1), (40000, 2), (300001, 3)])
def test_sample_small_weights_before_a_large_one(Q, gpu, V, seed, rules):
    """Tokens of 2^-50 to 2^-62 around and right before one of 1, by twos and fours of a lane, in other
    lanes, chunks and stretches: random numbers that fall on each of them."""
    g = torch.Generator().manual_seed(seed)
    last = V - 3
    x = torch.full((V,), -float("inf"))
    at = sorted({*range(last - 9, last), last + 1, *(int(V * torch.rand(1, generator=g)) for _ in range(24))} - {last})
    x[at] = -(50 + 12 * torch.rand(len(at), generator=g)) * math.log(2)
    x[last] = 0.0
    kept = sorted([*at, last])
    total = math.fsum(math.exp(float(x[i])) for i in kept)
    u, upto = [0.0], 0.0
    for i in kept[:kept.index(last)]:
        w = math.exp(float(x[i]))
        u += [(upto + w * v) / total for v in (0.01, 0.5, 0.99)]
        upto += w
    u += [upto * 1.01 / total, 0.5]
    check(Q, gpu, x, 1.0, u, kept, **rules)


def test_sample_of_a_large_weight_between_small_ones_by_chunks(Q, gpu):
    """Whole chunks of small weights, then one of 1 in a chunk of its own; thousands of tokens."""
    g = torch.Generator().manual_seed(9)
    for V, deep in ((40000, 55), (151936, 58)):
        x = -(deep + 4 * torch.rand(V, generator=g)) * math.log(2)
        last = V * 3 // 4
        x[last] = 0.0
        w = torch.exp(x.double())
        upto = torch.cumsum(w[:last], 0)
        total = float(w.sum())
        at = [1, 200, 255, 256, 3000, 10000, last - 1]
        u = torch.tensor([float(upto[i] - w[i] * 0.5) / total for i in at])
        for kw in (dict(), dict(min_p=torch.full((len(at),), 2.0 ** -63, device=gpu))):
            lp = torch.empty(len(at), device=gpu)
            got, _ = Q.sample(x.to(gpu).repeat(len(at), 1), u.to(gpu), logprob=lp, **kw)
            assert got.tolist() == at
            want = (x[at].double() - math.log(total)).to(gpu)
            assert ((lp - want).abs() <= 2.0 ** -24 * want.abs() + 1e-10).all()


@pytest.mark.parametrize("d,p", [(1.1291229724884033, 0.5224581956863403), (1.2371230125427246, 0.591297447681427)])
def test_sample_top_p_over_a_hundred_million_tokens(Q, gpu, d, p):
    """One token of 1 and 2^27 - 1 alike of w = exp(-d), where p times the whole sum lies 4 to 5 parts in
    10000 of w past a token's sum (2^-39 of the sum): the last token that is kept, by a random number
    whose token changes with it.  Sums within 2^-40 of a border may count as equal to it: 1.1 in 10000 here."""
    V = 1 << 27
    w = math.exp(-d)
    places = (p * (1 + (V - 1) * w) - 1) / w
    assert 3e-4 < places % 1 < 6e-4
    kept = 1 + (math.floor(places) + 1) * w
    u = next(v for v in (1 - i * 2.0 ** -24 for i in range(1, 200)) if 0.3 < (v * kept - 1) / w % 1 < 0.7)
    x = torch.full((1, V), -d, device=gpu)
    x[0, 0] = 0.0
    lp = torch.empty(1, device=gpu)
    got, _ = Q.sample(x, torch.tensor([u], device=gpu), top_p=torch.tensor([p], device=gpu), logprob=lp)
    assert int(got) == math.floor((u * kept - 1) / w) + 1
    assert abs(float(lp) - math.log(w / kept)) <= 2.0 ** -24 * 30 + 1e-10

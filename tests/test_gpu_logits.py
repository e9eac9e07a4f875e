"""q4k_logits_adjust against 64 bits: vocabularies of one token to several
slices, odd sizes and strides, empty lists and rows, repeated and foreign
tokens, masks that leave nothing."""
import pytest
import torch

import _batch

pytestmark = pytest.mark.gpu


def csr(lists, dtype, gpu):
    start = torch.tensor([0] + [len(x) for x in lists], dtype=torch.int64).cumsum(0).to(gpu)
    return torch.tensor([v for x in lists for v in x], dtype=dtype, device=gpu), start


def make(gpu, N, V, hist, nb, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, V, generator=g) * 4
    history = [(V * torch.rand(int(torch.randint(0, hist + 1, (1,), generator=g)), generator=g) ** 3).int().tolist() for _ in range(N)]
    biases = [[(int(t), float(b)) for t, b in zip(torch.randint(-2, V + 2, (nb,), generator=g), torch.randn(nb, generator=g) * 9)] for _ in range(N)]
    mask = torch.randint(-2 ** 31, 2 ** 31, (3, -(-V // 32)), generator=g).int()
    rows = torch.randint(-1, 4, (N,), generator=g).int()
    pen = [torch.rand(N, generator=g) + 0.8, torch.rand(N, generator=g), torch.rand(N, generator=g) - 0.5]
    return x.to(gpu), [p.to(gpu) for p in pen], history, biases, mask.to(gpu), rows.to(gpu)


def call(Q, gpu, x, pen, history, biases, mask, rows, **kw):
    h, hs = csr(history, torch.int32, gpu) if history is not None else (None, None)
    bi, bs = csr([[t for t, _ in r] for r in biases], torch.int32, gpu) if biases is not None else (None, None)
    bv = csr([[b for _, b in r] for r in biases], torch.float32, gpu)[0] if biases is not None else None
    return Q.logits_adjust(x, *pen, history=h, history_start=hs, bias_ids=bi, bias=bv, bias_start=bs, mask=mask, mask_rows=rows, **kw)


def check(Q, gpu, t, **kw):
    got = call(Q, gpu, *t, **kw)
    want, tol = _batch.logits(t[0], *t[1], t[2], t[3], t[4], t[5])
    _batch.assert_close(got, want, tol, "logits")
    return got


@pytest.mark.parametrize("N,V,hist,nb", [(1, 1, 3, 1), (1, 31, 5, 2), (3, 33, 40, 5), (2, 2048, 100, 0), (5, 2049, 700, 40),
                                        (1, 32768, 5000, 30), (9, 10007, 3000, 100), (20, 4100, 64, 3), (300, 257, 20, 2),
                                        (2, 151936, 9000, 300)])
def test_logits_sizes(Q, gpu, N, V, hist, nb):
    check(Q, gpu, make(gpu, N, V, hist, nb, seed=V))


def test_logits_parts_alone(Q, gpu):
    x, pen, history, biases, mask, rows = make(gpu, 4, 5000, 200, 10, 1)
    none = [None, None, None]
    assert torch.equal(call(Q, gpu, x, none, None, None, None, None), x)
    check(Q, gpu, (x, none, history, None, None, None))
    check(Q, gpu, (x, none, None, biases, None, None))
    check(Q, gpu, (x, none, None, None, mask, rows))
    check(Q, gpu, (x[:3], none, None, None, mask, None))
    for i in range(3):
        check(Q, gpu, (x, [p if j == i else None for j, p in enumerate(pen)], history, None, None, None))


def test_logits_last_bias_of_a_token_counts(Q, gpu):
    x = torch.zeros(2, 3000, device=gpu)
    biases = [[(5, 1.0), (2999, 4.0), (5, 2.0), (5, -3.0)], [(7, float("inf")), (9, -float("inf")), (7, 1.0)]]
    got = check(Q, gpu, (x, [None] * 3, None, biases, None, None))
    assert got[0, 5] == -3.0 and got[1, 7] == 1.0 and got[1, 9] == -float("inf")


def test_logits_foreign_tokens_and_backward_lists(Q, gpu):
    x, pen, _, _, _, _ = make(gpu, 3, 700, 10, 1, 2)
    check(Q, gpu, (x, pen, [[-1, 700, 3, 3, -2 ** 31, 2 ** 31 - 1], [], [699, 0]], [[(-1, 5.0)], [], [(700, 1.0), (1, 2.0)]], None, None))
    h = torch.arange(10, dtype=torch.int32, device=gpu)
    want = _batch.logits(x, *pen, [[], [3, 4], [0, 1, 2, 3, 4, 5, 6, 7, 8, 9][5:]], None, None, None)
    # starts that run backwards or past the list are empty or end with it
    for start in ([7, 3, 5, 10], [9, 3, 5, 99]):
        got = Q.logits_adjust(x, *pen, history=h, history_start=torch.tensor(start, device=gpu))
        _batch.assert_close(got, *want, "clamped lists")


def test_logits_masks_that_leave_nothing_or_everything(Q, gpu):
    x, pen, history, biases, _, _ = make(gpu, 3, 1000, 50, 5, 3)
    mask = torch.zeros(2, 40, dtype=torch.int32, device=gpu)
    mask[1] = -1
    rows = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
    got = check(Q, gpu, (x, pen, history, biases, mask, rows))
    assert (got[0] == -float("inf")).all()
    assert torch.isfinite(got[1:]).all()


def test_logits_special_values(Q, gpu):
    """NaN and infinities go through the arithmetic; the mask takes any of them out; zero counts as not positive."""
    x = torch.tensor([[float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e38, -1e38, 1e-40]], device=gpu)
    mask = torch.tensor([[0b11111110]], dtype=torch.int32, device=gpu)
    pen = [torch.tensor([2.0], device=gpu), None, None]
    got = call(Q, gpu, x, pen, [list(range(8))], None, mask, None)[0].tolist()
    assert got[0] == -float("inf") and got[1] == float("inf") and got[2] == -float("inf") and got[3] == 0 and got[4] == 0
    assert got[5] == 5e37 or abs(got[5] / 5e37 - 1) < 1e-6
    assert abs(got[6] / -2e38 - 1) < 1e-6
    got = call(Q, gpu, x, pen, [[0]], None, None, None)[0]
    assert torch.isnan(got[0]) and torch.equal(got[1:], x[0, 1:])


def test_logits_strides_in_place_and_odd_starts(Q, gpu):
    t = make(gpu, 6, 4999, 300, 20, 4)
    want = check(Q, gpu, t)
    nan = float("nan")
    for off, ooff in ((0, 0), (1, 1), (1, 2), (3, 0)):
        big = torch.full((6, 5011), nan, device=gpu)
        obig = torch.full((6, 5016), nan, device=gpu)
        x, out = big[:, off:off + 4999], obig[:, ooff:ooff + 4999]
        x.copy_(t[0])
        assert torch.equal(call(Q, gpu, x, *t[1:], out=out), want)
        assert torch.isnan(obig).sum() == 6 * (5016 - 4999)
        assert call(Q, gpu, x, *t[1:], out=x) is x and torch.equal(x, want)
        assert torch.isnan(big).sum() == 6 * (5011 - 4999)


def test_logits_graph(Q, gpu):
    x, pen, history, biases, mask, rows = make(gpu, 4, 9000, 400, 10, 6)
    h, hs = csr(history, torch.int32, gpu)
    out = torch.empty_like(x)
    args = dict(history=h, history_start=hs, mask=mask, mask_rows=rows)
    Q.logits_adjust(x, *pen, out=out, **args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        Q.logits_adjust(x, *pen, out=out, **args)
    for rep in range(4):
        x.normal_()
        h.copy_(torch.randint(0, 9000, h.shape, device=gpu))
        rows.copy_(torch.randint(-1, 3, rows.shape, device=gpu))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, Q.logits_adjust(x, *pen, **args)), rep


def test_logits_refusals_of_the_binding(Q, gpu):
    x = torch.zeros(2, 100, device=gpu)
    i32 = torch.zeros(2, dtype=torch.int32, device=gpu)
    with pytest.raises(ValueError):
        Q.logits_adjust(x.half())
    with pytest.raises(ValueError):
        Q.logits_adjust(x, history=i32)
    with pytest.raises(ValueError):
        Q.logits_adjust(x, repeat=torch.ones(3, device=gpu))
    with pytest.raises(ValueError):
        Q.logits_adjust(x, mask=torch.zeros(2, 3, dtype=torch.int32, device=gpu))
    with pytest.raises(ValueError):
        Q.logits_adjust(x, mask=torch.zeros(1, 4, dtype=torch.int32, device=gpu))
    assert Q.logits_adjust(x[:0]).shape == (0, 100)


def test_logits_list_starts_of_any_value(Q, gpu):
    """Starts so far apart that their difference passes 64 bits: the list is empty or ends with the entries there are."""
    lo, hi = -2 ** 63, 2 ** 63 - 1
    x, pen, _, _, _, _ = make(gpu, 7, 700, 10, 1, 2)
    h = torch.arange(10, dtype=torch.int32, device=gpu)
    bias = torch.arange(10, dtype=torch.float32, device=gpu)
    start = [5, lo, hi, lo, 3, hi, -9, 10 ** 15]
    lists = [list(range(10))[max(a, 0):max(b, 0)] for a, b in zip(start, start[1:])]
    assert [len(r) for r in lists] == [0, 10, 0, 3, 7, 0, 10]
    starts = torch.tensor(start, device=gpu)
    got = Q.logits_adjust(x, *pen, history=h, history_start=starts, bias_ids=h, bias=bias, bias_start=starts)
    want, tol = _batch.logits(x, *pen, lists, [[(t, float(t)) for t in r] for r in lists], None, None)
    _batch.assert_close(got, want, tol, "lists")

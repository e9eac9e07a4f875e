"""The operators of a decode step at sizes that a launch does not hold: refused as a whole, without an
error that a later call would report.  (Every size is that of real tensors or of a bound on them, so that
a launch would stay within them.)"""
import pytest
import torch

pytestmark = pytest.mark.gpu

EUNSUPPORTED = 1


def refused(Q, f, *args, **kw):
    with pytest.raises(Q.Q4KError) as e:
        f(*args, **kw)
    assert e.value.status == EUNSUPPORTED
    assert int(torch.ones(3, device="cuda:0").sum()) == 3  # (nobody else's call reports it)


@pytest.mark.parametrize("kv", [torch.int8, torch.float8_e4m3fn])
def test_bounds_on_a_requests_tokens_past_a_launch(Q, gpu, kv):
    hk, D = 2, 128
    t = [torch.ones(2, 16, hk, D, device=gpu).to(kv) for _ in range(2)] + [torch.full((2, 1, hk), 0.5, device=gpu) for _ in range(2)]
    pages, lens = Q.KV8Pages(*t), torch.tensor([16], dtype=torch.int32, device=gpu)
    start = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
    x = torch.full((1, hk, D), 2.0, device=gpu)
    out = torch.full((1, 4, D), 7.0, device=gpu)
    q = torch.randn(1, 4, D, device=gpu)
    want = Q.kv8_attention(q, pages, lens, 16, n_q=1, q_start=start)
    for n_q, ok in ((1 << 20, True), ((1 << 27) - 8, True), (1 << 27, False), ((1 << 30) - 1, False)):  # 2 x 128 / 8 threads a token
        y = x.clone()
        if ok:
            Q.kv8_load(pages, y, None, lens, 16, n_q=n_q, q_start=start)
            assert (y == 0.5).all()
        else:
            refused(Q, Q.kv8_load, pages, y, None, lens, 16, n_q=n_q, q_start=start)
            assert torch.equal(y, x)
    # (parts of four heads of 128 join eight rows a workgroup at most: 32 threads a row)
    assert torch.equal(Q.kv8_attention(q, pages, lens, 16, n_q=1 << 20, q_start=start, out=out), want)
    out.fill_(7.0)
    refused(Q, Q.kv8_attention, q, pages, lens, 16, n_q=1 << 28, q_start=start, out=out)
    assert (out == 7).all()
    refused(Q, Q.kv8_store, pages, x, x, lens, 16, n_q=(1 << 31) - 1, q_start=start)
    assert all((a.float() == 1).all() for a in t[:2])


def test_rows_and_tokens_past_a_launch(Q, gpu):
    n = 1 << 26
    for tokens, ok in ((n - 4, True), (n, False)):  # 64 threads each
        q = torch.ones(tokens, 1, 2, dtype=torch.float16, device=gpu)
        pos = torch.zeros(tokens, dtype=torch.int32, device=gpu)
        out = torch.zeros_like(q)
        if ok:
            Q.rope(Q.Rope(2), q, None, pos, q_out=out)
            assert torch.equal(out, q)
        else:
            refused(Q, Q.rope, Q.Rope(2), q, None, pos, q_out=out)
            assert not out.any()
    x = torch.zeros(1 << 23, 1, device=gpu)
    assert Q.sample_workspace(x).numel() == 16
    refused(Q, Q.sample, x)

"""q4k_rope against 64 bits: head sizes, parts of the head, layouts, scalings, far
positions, types, strides, in place, streams and graphs."""
import pytest
import torch

import _batch
import _step

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]
YARN = dict(freq_scale=0.25, ext_factor=1.0, n_ctx_orig=4096)


def inputs(gpu, n, H, hk, D, src, seed, far=5000):
    g = torch.Generator(device=gpu).manual_seed(seed)
    q, k = (torch.randn(n, h, D, device=gpu, generator=g).to(src) for h in (H, hk))
    return q, k, torch.randint(0, far + 1, (n,), device=gpu, generator=g).int(), g


def check(q, k, got, pos, D, n_rot, mode, q_norm=None, k_norm=None, base=10000.0, factors=None, yarn=None, what=""):
    kw = dict(freq_scale=yarn["freq_scale"], ext=yarn["ext_factor"], n_ctx=yarn["n_ctx_orig"]) if yarn else {}
    for name, x, y, w in (("q", q, got[0], q_norm), ("k", k, got[1], k_norm)):
        if x is None:
            assert y is None
            continue
        want, tol = _step.rope(x, pos, n_rot, mode, base=base, factors=factors, norm=w, out=y.dtype, **kw)
        _batch.assert_close(y, want, tol, f"{name} {what}")


@pytest.mark.parametrize("src,dst", TYPES)
@pytest.mark.parametrize("mode", ["normal", "neox"])
@pytest.mark.parametrize("n,H,hk,D,n_rot", [(1, 32, 8, 128, 128), (1, 1, 1, 2, 2), (3, 5, 1, 64, 64), (7, 24, 8, 80, 32), (65, 14, 2, 96, 48), (33, 8, 8, 256, 256),
                                            (130, 4, 4, 80, 20), (40, 3, 2, 250, 250), (9, 2, 1, 130, 6), (16, 6, 2, 64, 0)])
def test_rope_sizes(Q, gpu, src, dst, mode, n, H, hk, D, n_rot):
    q, k, pos, g = inputs(gpu, n, H, hk, D, src, n + D)
    outs = [torch.empty(x.shape, dtype=dst, device=gpu) for x in (q, k)]
    for norm in (False, True):
        w = [1 + 0.3 * torch.randn(D, device=gpu, generator=g) for _ in range(2)] if norm else [None, None]
        got = Q.rope(Q.Rope(D, n_rot=n_rot, mode=mode, q_norm=w[0], k_norm=w[1]), q, k, pos, q_out=outs[0], k_out=outs[1])
        assert got[0] is outs[0] and got[1] is outs[1]
        check(q, k, got, pos, D, n_rot, mode, *w, what=f"norm {norm}")


@pytest.mark.parametrize("mode", ["normal", "neox"])
@pytest.mark.parametrize("far", [1, 131072, 2 ** 31 - 1])
def test_rope_scalings_and_far_positions(Q, gpu, mode, far):
    for D, n_rot, base in ((128, 128, 500000.0), (80, 32, 10000.0), (64, 20, 1e6)):
        q, k, pos, g = inputs(gpu, 50, 4, 2, D, F32, D, far)
        pos[0], pos[1], pos[2] = 0, far, -far
        factors = 1 + 7 * torch.rand(n_rot // 2, device=gpu, generator=g)
        for kw in (dict(), dict(factors=factors), dict(yarn=YARN), dict(factors=factors, yarn=YARN)):
            r = Q.Rope(D, n_rot=n_rot, mode=mode, freq_base=base, freq_factors=kw.get("factors"), **kw.get("yarn", {}))
            check(q, k, Q.rope(r, q, k, pos), pos, D, n_rot, mode, base=base, what=str(sorted(kw)), **kw)


def test_rope_one_kind_and_norm_of_one_kind(Q, gpu):
    q, k, pos, g = inputs(gpu, 11, 6, 2, 64, F32, 1)
    w = 1 + 0.3 * torch.randn(64, device=gpu, generator=g)
    for qn, kn in ((w, None), (None, w)):
        r = Q.Rope(64, mode="neox", q_norm=qn, k_norm=kn)
        check(q, k, Q.rope(r, q, k, pos), pos, 64, 64, "neox", qn, kn)
        both = Q.rope(r, q, k, pos)
        assert torch.equal(Q.rope(r, q, None, pos)[0], both[0]) and torch.equal(Q.rope(r, None, k, pos)[1], both[1])
    # queries and keys of types of their own
    qo, ko = torch.empty_like(q, dtype=BF16), torch.empty_like(k)
    check(q, k, Q.rope(r, q, k, pos, q_out=qo, k_out=ko), pos, 64, 64, "neox", None, w)
    check(q.half(), k, Q.rope(r, q.half(), k, pos), pos, 64, 64, "neox", None, w)


@pytest.mark.parametrize("src", [F32, F16, BF16])
def test_rope_strides_alignment_and_in_place(Q, gpu, src):
    """Rows of a fused projection, places between rows left alone, odd addresses, in place."""
    n, H, hk, D = 37, 6, 2, 64
    for pad in (0, 1, 8):
        width = (H + 2 * hk) * D + pad
        g = torch.Generator(device=gpu).manual_seed(pad)
        base = torch.randn(n * width + 3, device=gpu, generator=g).to(src)
        for off in (0, 1):
            for mode in ("normal", "neox"):
                qkv = base.clone()[off:off + n * width].view(n, width)
                before = qkv.clone()
                q, k = qkv[:, :H * D].view(n, H, D), qkv[:, H * D:(H + hk) * D].view(n, hk, D)
                pos = torch.arange(n, device=gpu).int() * 3
                r = Q.Rope(D, n_rot=32, mode=mode)
                apart = Q.rope(r, q, k, pos)
                check(q, k, apart, pos, D, 32, mode)
                assert torch.equal(qkv, before)
                got = Q.rope(r, q, k, pos, q_out=q, k_out=k)
                assert got[0] is q and torch.equal(q, apart[0]) and torch.equal(k, apart[1])
                assert torch.equal(qkv[:, (H + hk) * D:], before[:, (H + hk) * D:])
    # heads that lie apart, tokens inside them
    x = torch.randn(4, 29, 64, device=gpu).to(src)
    pos = torch.arange(29, device=gpu).int()
    check(x.transpose(0, 1), None, Q.rope(Q.Rope(64), x.transpose(0, 1), None, pos), pos, 64, 64, "normal")


def test_rope_values_that_are_not_finite_stay_in_their_head(Q, gpu):
    q, k, pos, g = inputs(gpu, 5, 4, 2, 128, F32, 3)
    w = torch.ones(128, device=gpu)
    r = Q.Rope(128, mode="neox", q_norm=w, k_norm=w)
    want = Q.rope(r, q, k, pos)[0].clone()
    q[2, 1, 7] = float("nan")
    q[3, 0, 9] = float("inf")
    got = Q.rope(r, q, k, pos)[0]
    bad = torch.zeros(5, 4, dtype=torch.bool, device=gpu)
    bad[2, 1] = bad[3, 0] = True
    assert torch.equal(got[~bad], want[~bad]) and torch.isnan(got[2, 1]).all() and torch.isnan(got[3, 0, 9])


def test_rope_no_tokens_many_tokens_stream_and_graph(Q, gpu):
    r = Q.Rope(128, mode="neox", freq_base=500000.0)
    empty = Q.rope(r, torch.empty(0, 4, 128, device=gpu), torch.empty(0, 2, 128, device=gpu), torch.empty(0, dtype=torch.int32, device=gpu))
    assert empty[0].shape == (0, 4, 128)
    q, k, pos, g = inputs(gpu, 6000, 4, 1, 128, BF16, 5, 100000)
    want = Q.rope(r, q, k, pos)
    at = torch.randint(0, 6000, (64,), device=gpu, generator=g)
    check(q[at], k[at], [x[at] for x in want], pos[at], 128, 128, "neox", base=500000.0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = Q.rope(r, q, k, pos, stream=s)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a captured graph follows new positions
    out = [torch.empty_like(x) for x in (q, k)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        Q.rope(r, q, k, pos, q_out=out[0], k_out=out[1])
    for i in range(3):
        pos.copy_(torch.randint(0, 9999, (6000,), device=gpu, generator=g).int())
        graph.replay()
        torch.cuda.synchronize()
        want = Q.rope(r, q, k, pos)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        q.mul_(0.5)

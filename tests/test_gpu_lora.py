"""q4k_lora_add against 64 bits: token counts from one to several tiles, odd
sizes and ranks, strides, tokens without an adapter, ranks of zero, in place."""
import pytest
import torch

import _batch

pytestmark = pytest.mark.gpu


def make(gpu, N, K, M, r, A, dtype, seed, ids=None, ragged=False):
    g = torch.Generator(device=gpu).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=gpu, generator=g)  # noqa: E731
    a, b = (rnd(A, r, K) / max(K, 1) ** 0.5).to(dtype), rnd(A, M, r).to(dtype)
    if ids is None:
        ids = torch.randint(-1, A, (N,), device=gpu, generator=g).int()
    ranks = torch.randint(0, r + 2, (A,), device=gpu, generator=g).int() if ragged else None
    return a, b, rnd(N, K), ids, rnd(N, M), torch.rand(A, device=gpu, generator=g) - 0.3, ranks


def check(Q, t, **kw):
    a, b, x, ids, base, scale, ranks = t
    ad = Q.LoraAdapters(a, b, scale=scale, ranks=ranks)
    got = Q.lora_add(ad, x, ids, base=base, **kw)
    want, tol = _batch.lora(a, b, x, ids, base, scale, ranks)
    return _batch.assert_close(got, want, tol, "lora")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,K,M,r,A", [
    (1, 256, 64, 8, 1), (1, 4096, 1024, 16, 3), (2, 512, 100, 1, 2), (8, 4096, 1000, 16, 8), (7, 264, 33, 5, 3),
    (16, 1024, 256, 64, 2), (17, 999, 130, 13, 4), (33, 256, 17, 32, 40), (64, 2304, 513, 24, 5), (65, 768, 96, 40, 7),
    (130, 320, 1027, 96, 11), (300, 512, 200, 16, 3), (1025, 256, 128, 8, 70), (40, 640, 80, 256, 3), (5, 1, 1, 1, 2)])
def test_lora_sizes(Q, gpu, dtype, N, K, M, r, A):
    check(Q, make(gpu, N, K, M, r, A, dtype, seed=N + K))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,K,M,r,A", [(64, 8448, 130, 16, 1), (90, 8200, 96, 70, 2), (200, 8197, 64, 8, 3), (5000, 264, 64, 24, 300), (4097, 96, 36, 8, 1)])
def test_lora_long_sums_and_many_tokens(Q, gpu, dtype, N, K, M, r, A):
    check(Q, make(gpu, N, K, M, r, A, dtype, seed=N + K))


@pytest.mark.parametrize("N", [1, 9, 70, 200])
def test_lora_ranks_of_their_own(Q, gpu, N):
    check(Q, make(gpu, N, 512, 260, 24, 6, torch.float16, seed=N, ragged=True))


@pytest.mark.parametrize("N", [12, 150])
def test_lora_all_on_one_adapter_and_none(Q, gpu, N):
    one = torch.full((N,), 1, dtype=torch.int32, device=gpu)
    check(Q, make(gpu, N, 256, 128, 16, 3, torch.bfloat16, 1, ids=one))
    for none in (-1, 3, 2 ** 31 - 1, -2 ** 31):
        t = make(gpu, N, 256, 128, 16, 3, torch.bfloat16, 1, ids=torch.full_like(one, none))
        got = Q.lora_add(Q.LoraAdapters(t[0], t[1]), t[2], t[3], base=t[4])
        assert torch.equal(got, t[4])
        assert not Q.lora_add(Q.LoraAdapters(t[0], t[1]), t[2], t[3]).any()


def test_lora_long_runs_and_a_token_between(Q, gpu):
    """Prompts of one adapter each, as runs that do not end at tiles' ends."""
    ids = torch.cat([torch.full((n,), i) for n, i in ((100, 2), (1, 0), (63, 2), (65, 1), (31, -1), (129, 0))]).int().to(gpu)
    check(Q, make(gpu, ids.numel(), 384, 300, 16, 3, torch.float16, 5, ids=ids))


def test_lora_in_place_without_base_and_repeated_bits(Q, gpu):
    a, b, x, ids, base, scale, _ = make(gpu, 90, 1024, 520, 16, 7, torch.float16, 3)
    ad = Q.LoraAdapters(a, b, scale=scale)
    ws = Q.lora_workspace(ad, 90)
    ws.fill_(255)   # no initial contents needed
    want = Q.lora_add(ad, x, ids, base=base, workspace=ws)
    y = base.clone()
    assert Q.lora_add(ad, x, ids, base=y, out=y, workspace=ws) is y
    assert torch.equal(y, want)
    assert torch.equal(Q.lora_add(ad, x, ids, base=base), want)
    ref, tol = _batch.lora(a, b, x, ids, None, scale)
    _batch.assert_close(Q.lora_add(ad, x, ids), ref, tol, "no base")


def test_lora_strides_and_misaligned_rows(Q, gpu):
    """Rows apart, odd starts, one adapter read from a larger tensor: what is
    between the rows is neither read into the result nor written."""
    N, K, M, r, A = 70, 500, 300, 12, 5
    a, b, x, ids, base, scale, _ = make(gpu, N, K, M, r, A, torch.bfloat16, 9)
    nan = float("nan")
    def apart(t, off, pad):
        big = torch.full((*t.shape[:-1], t.shape[-1] + pad), nan, dtype=t.dtype, device=gpu)
        view = big[..., off:off + t.shape[-1]]
        view.copy_(t)
        return view
    want = Q.lora_add(Q.LoraAdapters(a, b, scale=scale), x, ids, base=base)
    outs = torch.full((N, M + 7), nan, device=gpu)
    for off in (1, 3, 8):
        out = outs[:, off - 1:off - 1 + M]
        t = (apart(a, off, 11), apart(b, off, 9), apart(x, off, 13), ids, apart(base, off % 4, 5), scale, None)
        assert check(Q, t, out=out) <= 1.0
        assert torch.isnan(outs).sum() == N * 7
        outs.fill_(nan)
    assert want.shape == (N, M)


def test_lora_large_activations_keep_f32_range(Q, gpu):
    a, b, x, ids, base, scale, _ = make(gpu, 20, 256, 64, 8, 2, torch.float16, 2)
    check(Q, (a, b, x * 1e12, ids, base, scale, None))
    check(Q, (a, b, x * 1e-12, ids, base * 0, scale, None))


def test_lora_infinite_activation_stays_with_its_token(Q, gpu):
    a, b, x, ids, base, scale, _ = make(gpu, 20, 256, 64, 8, 1, torch.float16, 2, ids=torch.zeros(20, dtype=torch.int32, device=gpu))
    ad = Q.LoraAdapters(a, b)
    want = Q.lora_add(ad, x, ids, base=base)
    x[7, 5] = float("nan")
    x[11, 3] = float("inf")
    got = Q.lora_add(ad, x, ids, base=base)
    keep = [i for i in range(20) if i not in (7, 11)]
    assert torch.equal(got[keep], want[keep])
    assert torch.isnan(got[7]).all() and not torch.isfinite(got[11]).any()


def test_lora_offsets_past_32_bits(Q, gpu):
    """Adapters more than 4 GiB apart."""
    K, M, r = 256, 64, 16
    gap = (1 << 31) + (1 << 20)
    big = torch.zeros(gap + M * K, dtype=torch.float16, device=gpu)
    a = big.as_strided((2, r, K), (gap, K, 1))
    b = big.as_strided((2, M, r), (gap, r, 1), r * K)
    g = torch.Generator(device=gpu).manual_seed(1)
    a.copy_(torch.randn(2, r, K, device=gpu, generator=g))
    b.copy_(torch.randn(2, M, r, device=gpu, generator=g))
    x = torch.randn(3, K, device=gpu, generator=g)
    ids = torch.tensor([1, 0, 1], dtype=torch.int32, device=gpu)
    got = Q.lora_add(Q.LoraAdapters(a, b), x, ids)
    want, tol = _batch.lora(a, b, x, ids)
    _batch.assert_close(got, want, tol, "far adapters")


def test_lora_graph_and_stream(Q, gpu):
    """A captured call follows ids, activations and base that change between replays."""
    for N in (8, 100):
        a, b, x, ids, base, scale, _ = make(gpu, N, 512, 256, 16, 5, torch.float16, 4)
        ad, out = Q.LoraAdapters(a, b, scale=scale), torch.empty_like(base)
        ws = Q.lora_workspace(ad, N)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            Q.lora_add(ad, x, ids, base=base, out=out, workspace=ws)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            Q.lora_add(ad, x, ids, base=base, out=out, workspace=ws)
        for rep in range(4):
            x.copy_(torch.randn_like(x))
            ids.copy_(torch.randint(-1, 5, (N,), device=gpu))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, Q.lora_add(ad, x, ids, base=base)), (N, rep)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        got = Q.lora_add(ad, x, ids, base=base, stream=s)
        s.synchronize()
        assert torch.equal(got, out)


def test_lora_refusals_of_the_binding(Q, gpu):
    a, b, x, ids, base, scale, _ = make(gpu, 4, 256, 64, 8, 2, torch.float16, 2)
    ad = Q.LoraAdapters(a, b)
    with pytest.raises(ValueError):
        Q.LoraAdapters(a, b.bfloat16())
    with pytest.raises(ValueError):
        Q.LoraAdapters(a, b, scale=scale[:1])
    with pytest.raises(ValueError):
        Q.lora_add(ad, x[:, :128], ids)
    with pytest.raises(ValueError):
        Q.lora_add(ad, x, ids.long())
    with pytest.raises(ValueError):
        Q.lora_add(ad, x, ids, base=base[:, ::2])
    with pytest.raises(Q.Q4KError):
        Q.lora_add(ad, x, ids, workspace=torch.empty(8, dtype=torch.uint8, device=gpu))
    assert Q.lora_add(ad, x[:0], ids[:0]).shape == (0, 64)


def test_lora_refuses_operands_in_host_memory(Q, gpu):
    a, b, x, ids, base, _, _ = make(gpu, 4, 256, 64, 8, 2, torch.float16, 2)
    ad = Q.LoraAdapters(a, b)
    size = Q.lora_workspace(ad, 4).numel()
    for bad in (dict(workspace=torch.empty(size, dtype=torch.uint8)), dict(workspace=torch.empty(1, dtype=torch.uint8, device=gpu).expand(size)),
                dict(base=base.cpu()), dict(out=torch.empty(4, 64))):
        with pytest.raises(ValueError):
            Q.lora_add(ad, x, ids, **bad)


@pytest.mark.parametrize("N,K,A", [(90, 333, 2), (300, 512, 30), (600, 333, 3), (600, 512, 40), (1500, 1024, 120)])
def test_lora_bits_do_not_depend_on_the_order_of_tokens(Q, gpu, N, K, A):
    """An adapter of 70 tokens, a tile of 64 and one of 6: whichever tokens come
    to lie in the second one have the same bits, from call to call too."""
    g = torch.Generator(device=gpu).manual_seed(N)
    ids = torch.randint(0, A, (N,), device=gpu, generator=g)
    ids[ids == 1] = -1
    ids[torch.randperm(N, device=gpu, generator=g)[:70]] = 1
    a, b, x, ids, base, scale, _ = make(gpu, N, K, 64, 16, A, torch.float16, seed=N, ids=ids.int())
    ad = Q.LoraAdapters(a, b, scale=scale)
    want = Q.lora_add(ad, x, ids, base=base)
    for _ in range(3):
        perm = torch.randperm(N, device=gpu, generator=g)
        assert torch.equal(Q.lora_add(ad, x[perm], ids[perm], base=base[perm]), want[perm])
        assert torch.equal(Q.lora_add(ad, x, ids, base=base), want)


@pytest.mark.parametrize("A,K,most,N", [(256, 4096, 254, 127), (16, 4096, 1024, 1023), (4, 14336, 896, 895), (3, 4096, 600, 1)])
def test_lora_workspace_of_a_larger_batch(Q, gpu, A, K, most, N):
    a, b, x, ids, base, scale, _ = make(gpu, N, K, 64, 16, A, torch.float16, seed=N)
    ad = Q.LoraAdapters(a, b, scale=scale)
    got = Q.lora_add(ad, x, ids, base=base, workspace=Q.lora_workspace(ad, most))
    assert torch.equal(got, Q.lora_add(ad, x, ids, base=base, workspace=Q.lora_workspace(ad, N)))


@pytest.mark.parametrize("N", [1, 40, 700])
def test_lora_adapters_that_add_nothing(Q, gpu, N):
    """No rank or no activations: the base, whatever scale (alpha over a rank of zero) and b hold."""
    inf, nan = float("inf"), float("nan")
    a, b, x, _, base, _, _ = make(gpu, N, 256, 96, 8, 3, torch.float16, 1)
    ids = torch.arange(N, dtype=torch.int32, device=gpu) % 2 * 2
    scale, ranks = torch.tensor([inf, 1.0, nan], device=gpu), torch.tensor([0, 8, -1], dtype=torch.int32, device=gpu)
    b[0], b[2] = inf, nan
    assert torch.equal(Q.lora_add(Q.LoraAdapters(a, b, scale=scale, ranks=ranks), x, ids, base=base), base)
    assert torch.equal(Q.lora_add(Q.LoraAdapters(a[:, :, :0], b, scale=scale), x[:, :0], ids, base=base), base)
    empty = torch.empty(3, 8, 0, dtype=torch.float16, device=gpu)
    assert torch.equal(Q.lora_add(Q.LoraAdapters(empty, b, scale=scale), torch.empty(N, 0, device=gpu), ids, base=base), base)

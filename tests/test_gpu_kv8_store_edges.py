"""q4k_kv8_store where a block has nothing that a scale could be taken from."""
import pytest
import torch

import _step

pytestmark = pytest.mark.gpu

I8, E4M3 = torch.int8, torch.float8_e4m3fn


@pytest.mark.parametrize("kind", [I8, E4M3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,block,n", [(16, 1, 3), (64, 16, 48), (128, 32, 96), (256, 64, 192), (80, 100, 300)])
def test_store_infinities_alone(Q, gpu, kind, dtype, D, block, n):
    """Blocks of infinities and zeros, infinities and NaN, NaN alone, zeros alone: infinities read
    back as the largest of their sign, the rest as 0; with a finite value beside them, by its scale."""
    inf, nan, top = float("inf"), float("nan"), _step.TOP[kind]
    for at in (0, block // 2, block - 1):
        t = [torch.full((n // block, block, 2, D), 3, device=gpu).to(kind) for _ in range(2)] + [torch.full((n // block, 1, 2), 0.25, device=gpu) for _ in range(2)]
        k, v = (torch.zeros(n, 2, D, device=gpu) for _ in range(2))
        first = k[:block]
        first[at, 0, D - 1], first[0, 0, 0], first[at, 1] = inf, -inf, nan
        v[block:2 * block, 1] = nan
        v[block + at, 1, D // 2] = -inf
        v[2 * block + at, 0, 1], v[2 * block, 0, 0] = inf, -0.5
        pages = Q.KV8Pages(*t, table=torch.arange(n // block, device=gpu).int()[None])
        lens = torch.tensor([n], dtype=torch.int32, device=gpu)
        Q.kv8_store(pages, k.to(dtype), v.to(dtype), lens, n, n_q=n)
        got = [torch.empty(n, 2, D, device=gpu) for _ in range(2)]
        Q.kv8_load(pages, *got, lens, n, n_q=n)
        scale = torch.tensor(0.5).double().div(top).float()
        for x, y, s in ((k, got[0], t[2]), (v, got[1], t[3])):
            want = torch.nan_to_num(x, nan=0.0, posinf=top, neginf=-top)
            if x is v:
                want[2 * block:, 0] = torch.where(torch.isinf(x[2 * block:, 0]), top * scale.to(gpu), want[2 * block:, 0])
                want[2 * block, 0, 0] = -top * scale
                assert s[2, 0, 0] == scale.to(gpu) and s[1, 0, 1] == 1 and s[1, 0, 0] == 0
            else:
                assert s[0, 0, 0] == 1 and s[0, 0, 1] == 0 and not s[1:].any()
            assert torch.equal(y, want)


@pytest.mark.parametrize("kind", [I8, E4M3])
def test_store_infinities_before_and_after_finite_values(Q, gpu, kind):
    """Token by token in one block: zeros, an infinity, small values, larger ones."""
    inf, top = float("inf"), _step.TOP[kind]
    t = [torch.zeros(1, 8, 1, 16, device=gpu).to(kind) for _ in range(2)] + [torch.full((1, 1, 1), 9.0, device=gpu) for _ in range(2)]
    pages = Q.KV8Pages(*t)
    for step, (value, scale, reads) in enumerate([
            (0.0, 0.0, [0.0]), (inf, 1.0, [0.0, top]), (3.0, 1.0, [0.0, top, 3.0]), (-inf, 1.0, [0.0, top, 3.0, -top]),
            (4 * top, 4.0, [0.0, top, 4.0 if kind == I8 else 3.0, -top, 4 * top])]):
        x = torch.full((1, 1, 16), value, device=gpu)
        lens = torch.tensor([step + 1], dtype=torch.int32, device=gpu)
        Q.kv8_store(pages, x, -x, lens, 8)
        got = [torch.empty(step + 1, 1, 16, device=gpu) for _ in range(2)]
        Q.kv8_load(pages, *got, lens, 8, n_q=step + 1)
        assert float(t[2]) == float(t[3]) == scale
        want = torch.tensor(reads, device=gpu)
        if kind == I8 and step == 4:
            want[1], want[3] = 128.0, -128.0  # 127 of a scale of 4: the nearest is 32
        assert torch.equal(got[0][:, 0, 3], want) and torch.equal(got[1][:, 0, 3], -want)

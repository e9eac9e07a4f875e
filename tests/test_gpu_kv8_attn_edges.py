"""q4k_kv8_attn where several of its rare cases meet, against 64 bits."""
import pytest
import torch

import _batch
import _batch_terms
from test_gpu_kv8_attn import BF16, E4M3, F16, F32, I8, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("qt", [F32, F16, BF16])
@pytest.mark.parametrize("block", [8, 4])
@pytest.mark.parametrize("B,nq,most", [(2, 1, 300), (2, 3, 300), (40, 1, 1300)])
def test_kv8_attention_nan_beside_a_missing_page(Q, gpu, qt, block, B, nq, most):
    """A value of NaN and a page out of range within the same 32 positions, which every query sees,
    at each place of the step: the queries get the NaN, as without the missing page."""
    for place in range(4):
        c = Case(gpu, B, nq, 4, 2, 64, most, 8, block, qt, E4M3, seed=place, lens=[most] * B)
        j, missing = 64 + 8 * place + 3, 64 + 8 * ((place + 1) % 4)
        for r in range(0, B, 7):
            for d, head in ((5, 0), (63, 1)):
                c.t[1].view(torch.uint8)[int(c.table[r, j // 8]), j % 8, head, d] = 0x7f if d == 5 else 0xff
            c.table[r, missing // 8] = -1 if place % 2 else 10 ** 6
        out, lse = c.check(Q)
        bad = torch.isnan(out)
        assert bad[:nq, :2, 5].all() and bad[:nq, 2:, 63].all() and int(bad.sum()) == nq * 4 * len(range(0, B, 7)) and lse.isfinite().all()


@pytest.mark.parametrize("kv", [I8, E4M3])
@pytest.mark.parametrize("B,H,hk,D", [(3, 8, 2, 128), (5, 4, 4, 256), (9, 3, 1, 80), (2, 6, 3, 64)])
@pytest.mark.parametrize("above", [0, 5, 10, 14, 17, 20, 24])
def test_kv8_attention_scores_keep_f32_beside_a_larger_value(Q, gpu, kv, B, H, hk, D, above):
    """One key, and a query of one value that meets it and one 2^above larger that meets a zero: the
    log-sum-exp is the score, at the bound of a query of that value alone down to 2^-17 of the
    larger one, below that with 2^-39 of it for the query's last bit."""
    U = _batch_terms.U
    g = torch.Generator(device=gpu).manual_seed(above)
    for magnitude in (0, -60, 60):
        at = torch.randint(0, D, (B, H), device=gpu, generator=g)
        other = (at + torch.randint(1, D, (B, H), device=gpu, generator=g)) % D
        value = _batch_terms.full((B, H), g, gpu, 3, 6)
        larger = value.abs() * 2.0 ** above * (1 + torch.rand(B, H, device=gpu, generator=g))
        q = torch.zeros(B, H, D, device=gpu).scatter_(2, other[:, :, None], larger[:, :, None]).scatter_(2, at[:, :, None], value[:, :, None])
        k = torch.randint(1, 120, (B, 16, hk, D), device=gpu, generator=g).float()
        k = k.repeat_interleave(H // hk, 2).scatter_(3, other[:, None, :, None].expand(B, 16, H, 1), 0.0).to(kv)  # (a head of keys a query)
        s = [torch.rand(B, 1, hk, device=gpu, generator=g).repeat_interleave(H // hk, 2) * 0.01 + 0.005 for _ in range(2)]
        lse = torch.empty(B, H, device=gpu)
        Q.kv8_attention(q * 2.0 ** magnitude, Q.KV8Pages(k, k, *s), torch.ones(B, dtype=torch.int32, device=gpu), 16, scale=2.0 ** -magnitude, lse=lse)
        kd = (k[:, 0].float().double() * s[0].double().transpose(1, 2)).gather(2, at[:, :, None])[:, :, 0]
        want = value.double() * kd
        tol = 10 * U * want.abs() + 2.0 ** -18 + 2.0 ** -39 * larger.double() * kd
        _batch.assert_close(lse, want.cpu(), tol.cpu(), f"score, 2^{above}, magnitude 2^{magnitude}")

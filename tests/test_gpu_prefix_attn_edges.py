"""q4k_prefix_attn: F32 queries of values far apart."""
import pytest
import torch

import _batch
import _batch_terms

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,H,D", [(3, 8, 128), (70, 4, 128), (5, 4, 256), (9, 3, 80), (130, 6, 64)])
@pytest.mark.parametrize("above", [0, 5, 10, 14, 17, 20, 24])
def test_attention_scores_keep_f32_beside_a_larger_value(Q, gpu, kv, B, H, D, above):
    """One key, and queries of one value that meets it and one 2^above larger that meets a zero: the
    log-sum-exp is the score, at the bound of a query of that value alone down to 2^-17 of the
    larger one, below that with 2^-39 of it for the query's last bit."""
    U = _batch_terms.U
    g = torch.Generator(device=gpu).manual_seed(above)
    for magnitude in (0, -60, 60):
        at = torch.randint(0, D, (H,), device=gpu, generator=g)
        other = (at + torch.randint(1, D, (H,), device=gpu, generator=g)) % D
        value = _batch_terms.full((B, H), g, gpu, 3, 6)
        larger = value.abs() * 2.0 ** above * (1 + torch.rand(B, H, device=gpu, generator=g))
        h = torch.arange(H, device=gpu)
        q = torch.zeros(B, H, D, device=gpu)
        q[:, h, other] = larger
        q[:, h, at] = value
        k = torch.randn(1, 1, H, D, device=gpu, generator=g)
        k[0, 0, h, other] = 0.0
        k = k.to(kv)
        lse = torch.empty(B, H, device=gpu)
        Q.prefix_attention(q * 2.0 ** magnitude, Q.KVPages(k, k, table=torch.zeros(1, dtype=torch.int32, device=gpu)), 1, scale=2.0 ** -magnitude, lse=lse)
        kd = k[0, 0, h, at].double()
        want = value.double() * kd
        tol = 10 * U * want.abs() + 2.0 ** -18 + 2.0 ** -39 * larger.double() * kd.abs()
        _batch.assert_close(lse, want.cpu(), tol.cpu(), f"score, 2^{above}, magnitude 2^{magnitude}")

"""q4k_kv8_attn where several of its rare cases meet, against 64 bits."""
import pytest
import torch

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

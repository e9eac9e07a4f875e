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

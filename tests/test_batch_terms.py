"""The bounds of _batch_terms.py on the CPU: arithmetic with the stated terms
keeps them, and without the smallest term of any value it does not."""
import pytest
import torch

import _batch_terms as T

F16, BF16 = torch.float16, torch.bfloat16


def split(x, dtype, n):
    """x as the sum of n values of dtype, in 64 bits."""
    out, r = [], x.double()
    for _ in range(n):
        out.append(r.to(dtype).double())
        r = r - out[-1]
    return out


def product(w, x, drop):
    """The adapters' product: w of 16 bits times F32 x, without the term `drop`."""
    wt, xt = split(w, BF16, 2 if w.dtype == F16 else 1), split(x, BF16, 3)
    keep = [(i, j) for i in range(len(wt)) for j in range(3) if i + j < 3 and (i, j) != drop]
    return sum(wt[i] * xt[j] for i, j in keep).float()


def lora(a, b, x, ids, base, scale, drop=(None, None)):
    N, at = x.shape[0], x.abs().argmax(1)
    n, m = torch.arange(N), torch.arange(b.shape[1])
    ids = ids.long()
    h = product(a[ids, :, at], x[n, at][:, None], drop[0])
    j = m % a.shape[1]
    return base + product(b[:, m, j][ids], (h * scale[ids][:, None])[:, j], drop[1])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_adapters_bound(dtype):
    *t, want, tol = T.lora_inputs("cpu", 40, 64, 90, 16, 3, dtype, 1)
    assert ((lora(*t) - want).abs() <= tol).all()
    smallest = [(0, 2)] + ([(1, 1), (1, 0)] if dtype == F16 else [])
    for term in smallest:
        for drop in ((term, None), (None, term)):
            assert ((lora(*t, drop=drop) - want).abs() > tol).any(), drop


def attention(q, k, v, kv, terms_q, terms_p):
    """Scores and probabilities in F32 with the terms given; (out, lse)."""
    grp = q.shape[1] // k.shape[1]
    kd, vd = (t.double().repeat_interleave(grp, 1) for t in (k, v))
    top = q.abs().amax(2, keepdim=True)
    f = torch.exp2(-torch.floor(torch.log2(top)))
    qs = sum(split(q * f, kv, terms_q)) / f.double()
    s = torch.einsum("bhd,nhd->bhn", qs, kd).float()
    m = s.amax(2, keepdim=True)
    p = torch.exp((s - m).double()).float() * 128
    total = p.sum(2, keepdim=True)
    out = torch.einsum("bhn,nhd->bhd", sum(split(p, kv, terms_p)), vd).float() / total
    return out, (m + torch.log(total / 128))[:, :, 0]


@pytest.mark.parametrize("kv,terms", [(F16, 2), (BF16, 3)])
def test_attention_bounds(kv, terms):
    q, k, v, want, tol = T.score_inputs("cpu", 9, 8, 2, 64, kv, 2)
    assert ((attention(q, k, v, kv, terms, terms)[1] - want).abs() <= tol).all()
    assert ((attention(q, k, v, kv, terms - 1, terms)[1] - want).abs() > tol).any()
    q, k, v, want, tol = T.probability_inputs("cpu", 9, 8, 2, 64, 50, kv, 3)
    assert ((attention(q, k, v, kv, terms, terms)[0] - want).abs() <= tol).all()
    assert ((attention(q, k, v, kv, terms, terms - 1)[0] - want).abs() > tol).any()

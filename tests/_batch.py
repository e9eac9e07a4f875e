"""64-bit references of the batch operators, on the CPU, and error bounds that
follow from the operators' stated roundings (include/q4k_batch.h)."""
from __future__ import annotations

import torch

U16 = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a unit in the last place, relative


def lora(a, b, x, ids, base=None, scale=None, ranks=None):
    """(result, bound).  The activations and h hold 16 bits or more each (2^-16
    of every term), the F32 sums a part of that; adding the base rounds once."""
    a, b, x = a.double().cpu(), b.double().cpu(), x.double().cpu()
    N, M = x.shape[0], b.shape[1]
    out = base.double().cpu().clone() if base is not None else torch.zeros(N, M, dtype=torch.float64)
    l1 = torch.zeros(N, M, dtype=torch.float64)
    for n, i in enumerate(ids.tolist()):
        if not 0 <= i < a.shape[0]:
            continue
        r = a.shape[1] if ranks is None else min(max(int(ranks[i]), 0), a.shape[1])
        s = 1.0 if scale is None else float(scale[i])
        out[n] += s * (b[i, :, :r] @ (a[i, :r] @ x[n]))
        l1[n] = abs(s) * (b[i, :, :r].abs() @ (a[i, :r].abs() @ x[n].abs()))
    return out, 2.0 ** -15 * l1 + 2.0 ** -22 * out.abs() + 1e-30


def kv_of(k, v, table, length, heads_kv, dim):
    """The first `length` tokens of one request, and which of them have a page."""
    page = k.shape[1]
    at = torch.arange(length)
    pages = table.long().cpu()[at // page]
    ok = (pages >= 0) & (pages < k.shape[0])
    pages = torch.where(ok, pages, 0)
    return k.cpu()[pages, at % page].double(), v.cpu()[pages, at % page].double(), ok


def attention(q, spans, prefix, suffix, lens, scale):
    """spans: the [first, last) tokens of each request; prefix, suffix:
    (k, v, tables of page numbers) or None; lens: (prefix tokens, tokens of each
    request).  Returns (out, lse, bound of out, bound of lse)."""
    H, D = q.shape[1], q.shape[2]
    some = prefix or suffix
    hk, kv = some[0].shape[2], some[0].dtype
    u = 2.0 ** -15 if q.dtype == torch.float32 else U16[kv]   # of a probability
    uo = 2.0 ** -23 if q.dtype == torch.float32 else U16[kv]  # of the stored result
    qd = q.double().cpu()
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -float("inf"), dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for r, (t0, t1) in enumerate(spans):
        parts = []
        if lens[0]:
            parts.append(kv_of(*prefix[:2], prefix[2], lens[0], hk, D))
        if lens[1] is not None and lens[1][r] > 0:
            parts.append(kv_of(*suffix[:2], suffix[2][r], lens[1][r], hk, D))
        if not parts:
            continue
        k, v, ok = (torch.cat([p[i] for p in parts]) for i in range(3))
        for t in range(t0, t1):
            seen = ok.clone()
            own = 0 if lens[1] is None else max(lens[1][r], 0)
            last = lens[0] + own - (t1 - t0) + (t - t0)
            seen[max(lens[0], last + 1):] = False
            if not seen.any():
                continue
            ks = k[seen].repeat_interleave(H // hk, 1)
            vs = v[seen].repeat_interleave(H // hk, 1)
            s = (ks * qd[t]).sum(-1) * scale                                    # [L, H]
            e = (ks.abs() * qd[t].abs()).sum(-1).amax(0) * abs(scale) * 2.0 ** -17
            lse[t] = torch.logsumexp(s, 0)
            p = torch.softmax(s, 0)
            out[t] = (p[:, :, None] * vs).sum(0)
            mass = (p[:, :, None] * vs.abs()).sum(0)
            tol[t] = (1.5 * u + 2 * e[:, None]) * mass + 2.0 ** -24 * vs.abs().sum(0) / torch.exp(lse[t] - s.amax(0))[:, None] \
                + uo * out[t].abs() + 1e-30
            tol_lse[t] = 2 * e + 2.0 ** -18 + 2.0 ** -21 * lse[t].abs()
    return out, lse, tol, tol_lse


def logits(x, repeat, frequency, presence, history, biases, mask, mask_rows):
    """history: a list of tokens a row; biases: a list of (token, bias) a row.  (result, bound)"""
    # every step rounds to F32: 2^-24 of what it adds up, and of the stored result
    out = x.double().cpu().clone()
    V = out.shape[1]
    mag = torch.zeros_like(out)
    for i in range(out.shape[0]):
        get = lambda t, d: d if t is None else float(t[i])  # noqa: E731
        p, f, s = get(repeat, 1.0), get(frequency, 0.0), get(presence, 0.0)
        count = {}
        for t in history[i] if history else []:
            if 0 <= t < V:
                count[t] = count.get(t, 0) + 1
        for t, c in count.items():
            y = out[i, t] / p if out[i, t] > 0 else out[i, t] * p
            mag[i, t] += y.abs() + abs(c * f) + abs(s)
            out[i, t] = y - c * f - s
        for t, b in dict(biases[i] if biases else []).items():
            if 0 <= t < V:
                out[i, t] += b
                mag[i, t] += abs(b)
        if mask is not None:
            m = i if mask_rows is None else int(mask_rows[i])
            if 0 <= m < mask.shape[0]:
                at = torch.arange(V)
                out[i, ((mask[m].cpu()[at // 32] >> (at % 32)) & 1) == 0] = -float("inf")
    touched = torch.where(torch.isfinite(out) & (mag > 0), out.abs(), 0.0)
    return out, 2.0 ** -22 * mag + 2.0 ** -23 * touched


def assert_close(got, want, tol, what):
    """Elementwise within the bound; infinities and NaN in the same places."""
    got = got.double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN elsewhere"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), f"{what}: infinities"
    err = torch.where(fine, (got - want).abs(), 0.0)
    bad = fine & ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, worst {float((err / tol)[bad].max()):.3g} times at {bad.nonzero()[0].tolist()}"
    return float((err[fine] / tol[fine].clamp(min=1e-300)).max()) if fine.any() else 0.0

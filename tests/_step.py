"""64-bit references of the operators of a decode step (include/q4k_step.h), on
the CPU, and error bounds from the roundings that the header states."""
from __future__ import annotations

import math

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def rope(x, pos, n_rot, mode, base=10000.0, freq_scale=1.0, ext=0.0, attn=1.0, fast=32.0, slow=1.0, n_ctx=0, factors=None, norm=None,
         eps=1e-6, out=None):
    """(result, bound) of one kind of rows x [tokens, heads, dim].

    The bound: of a normed value, the sum of squares of up to 256 terms (at most 64
    F32 roundings one after the other in any order that the kernel may take, halved
    by the root), the root, the quotient and two products: 40 units of 2^-24.  A rotation adds
    two products and a sum (3 units of |a| + |b|) and its cosines: a quarter turn's
    rest rounded to F32 (2^-25 of up to pi / 4 radians), the functions' own units (2)
    and the magnitude's (1).  Then one rounding to the type."""
    x = x.double().cpu()
    mag, u = torch.zeros_like(x), 2.0 ** -24
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * norm.double().cpu()
        mag = 40 * u * x.abs()
    y = x.clone()
    lo, hi = 0.0, 0.0
    if ext:
        lo, hi = (0.5 * n_rot * math.log(n_ctx / (b * 2 * math.pi)) / math.log(base) for b in (fast, slow))
        lo, hi = max(0, math.floor(lo)), min(n_rot - 1, math.ceil(hi))
    for i in range(n_rot // 2):
        f, m = base ** (-2 * i / n_rot), attn
        if factors is not None:
            f /= float(factors[i])
        if ext:
            r = ext * (1 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo))))
            f *= freq_scale * (1 - r) + r
            m *= 1 + 0.1 * math.log(1 / freq_scale)
        else:
            f *= freq_scale
        t = (pos.double().cpu() * f)[:, None]
        a, b = (2 * i, 2 * i + 1) if mode == "normal" else (i, i + n_rot // 2)
        y[..., a] = m * (x[..., a] * t.cos() - x[..., b] * t.sin())
        y[..., b] = m * (x[..., a] * t.sin() + x[..., b] * t.cos())
        both = abs(m) * (x[..., a].abs() + x[..., b].abs())
        # (64-bit angles: the power's and the product's units, of turns, in both)
        far = pos.double().abs().cpu()[:, None] * f * 2.0 ** -46
        tol = both * (10 * u + far) + abs(m) * (mag[..., a] + mag[..., b])
        mag[..., a], mag[..., b] = tol, tol
    return y, mag + UNIT[out or torch.float32] * y.abs() * (1 + 2.0 ** -8) + 1e-38 + (2.0 ** -25 if out == torch.float16 else 0)


# ------------------------------------------------------------ caches of 8 bits ----
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
#: every value of e4m3 from 0 up, by its code
CODES = torch.tensor([m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127],
                     dtype=torch.float64)


def round8(x, scale, dtype):
    """x / scale in 64 bits to the nearest value of dtype (as its bytes' values, float64),
    ties to even; x F32, scale F32 of x's shape."""
    y = x.double() / torch.where(scale > 0, scale, 1.0).double()
    y = torch.where(scale > 0, y, 0.0)
    y = torch.where(torch.isinf(x), x.double(), y)
    y = torch.where(torch.isnan(x), 0.0, y).clamp(-TOP[dtype], TOP[dtype])
    if dtype == torch.int8:
        return torch.round(y)
    mid = (CODES[1:] + CODES[:-1]) / 2
    i = torch.searchsorted(mid, y.abs().contiguous())
    i = i + ((y.abs() == mid[i.clamp(max=125)]) & (i % 2 == 1)).long()
    return torch.sign(y) * CODES[i]


class Cache8:
    """A cache of 8 bits in plain steps on the CPU: bytes' values [pages, page, heads, dim] float64, scales F32."""

    def __init__(self, k, v, k_scale, v_scale, table):
        self.dtype = k.dtype
        self.held = [t.cpu().float().double() for t in (k, v)]
        self.scale = [t.cpu().clone() for t in (k_scale, v_scale)]
        self.table, self.page = table.long().cpu(), k.shape[1]
        self.block = self.page // k_scale.shape[1]

    def place(self, r, t):
        p = int(self.table[r, t // self.page])
        return (p, t % self.page) if 0 <= p < self.held[0].shape[0] else None

    def store(self, new, spans, lens):
        """new: (k, v) rows; spans: [first, last) tokens of a request."""
        for r, (t0, t1) in enumerate(spans):
            first = lens[r] - (t1 - t0)
            for b0 in sorted({t // self.block * self.block for t in range(max(first, 0), lens[r])}):
                at = self.place(r, b0)
                if at is None:
                    continue
                p, s0 = at
                lo, hi = max(first, b0), min(lens[r], b0 + self.block)
                for held, scale, x in zip(self.held, self.scale, new):
                    rows = x[t0 + lo - first:t0 + hi - first].float().cpu()           # [n, heads, dim]
                    top = torch.where(torch.isfinite(rows), rows.abs(), 0.0).amax((0, 2))
                    s = (top.double() / TOP[self.dtype]).float()
                    was = scale[p, s0 // self.block]
                    if lo > b0:
                        s = torch.maximum(s, was)
                        old = held[p, s0:s0 + lo - b0]
                        again = round8((old * was.double()[:, None]).float(), s[:, None].expand(old.shape), self.dtype)
                        held[p, s0:s0 + lo - b0] = torch.where((s > was)[:, None], again, old)
                    held[p, s0 + lo - b0:s0 + hi - b0] = round8(rows, s[:, None].expand(rows.shape), self.dtype)
                    scale[p, s0 // self.block] = s

    def values(self, r, length):
        """Keys and values of the first tokens of a request, float64, and which have a page."""
        at = torch.arange(length)
        pages = self.table[r][at // self.page]
        ok = (pages >= 0) & (pages < self.held[0].shape[0])
        pages = torch.where(ok, pages, 0)
        s = at % self.page
        return [h[pages, s] * c[pages, s // self.block].double()[:, :, None] for h, c in zip(self.held, self.scale)] + [ok]


# ------------------------------------------------ attention over caches of 8 bits ----
#: what a probability times its value's scale keeps: terms of BF16, three and two
PROBABILITY = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -15, torch.bfloat16: 2.0 ** -15}


def attention8(q, spans, cache, lens, scale):
    """(out, lse, bound of out, bound of lse) of queries q [tokens, heads, dim], the
    spans' [first, last) tokens of each request, over a Cache8.

    The bounds: a score is off by e, 2^-17 of sum |q k| (two F16 terms of a query
    2^-22 of each product, F32 sums of up to 256 of them and their scale and factor
    below 64 units of 2^-24); a probability by 2 e, the exponent's units (2^-22) and what
    its terms keep; a sum over n positions by a unit for each step of a wave (n /
    128) and 40 more for its lanes, waves and splits."""
    H, D = q.shape[1], q.shape[2]
    hk = cache.held[0].shape[2]
    u, uo = PROBABILITY[q.dtype], UNIT[q.dtype]
    qd = q.double().cpu()
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -float("inf"), dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for r, (t0, t1) in enumerate(spans):
        length = max(0, lens[r])
        k, v, ok = cache.values(r, length)
        for t in range(t0, t1):
            seen = ok.clone()
            seen[max(0, length - (t1 - t0) + (t - t0) + 1):] = False
            if not seen.any():
                continue
            ks = k[seen].repeat_interleave(H // hk, 1)
            vs = v[seen].repeat_interleave(H // hk, 1)
            s = (ks * qd[t]).sum(-1) * scale                                    # [L, H]
            e = (ks.abs() * qd[t].abs()).sum(-1).amax(0) * abs(scale) * 2.0 ** -17 + 2.0 ** -22
            lse[t] = torch.logsumexp(s, 0)
            p = torch.softmax(s, 0)
            out[t] = (p[:, :, None] * vs).sum(0)
            mass = (p[:, :, None] * vs.abs()).sum(0)
            sums = (s.shape[0] / 128 + 40) * 2.0 ** -24
            tol[t] = (u + 2 * e[:, None] + 2 * sums) * mass + uo * out[t].abs() * 1.01 + 1e-30
            tol_lse[t] = 2 * e + 2 * sums + 2.0 ** -21 * lse[t].abs()
            if q.dtype == torch.float16:
                tol[t] += 2.0 ** -25
    return out, lse, tol, tol_lse


# --------------------------------------------------------------------- next tokens ----
def sample(logits, u, t, k, p, m):
    """(token, log-probability, margin) of one row in 64 bits: the margin is how far, of
    the kept or the whole sum, the nearest other choice lies (a kernel whose sums
    are of 64 bits too decides alike beyond some 2^-40 of it)."""
    x = logits.double().cpu()
    x = torch.where(torch.isnan(x), -float("inf"), x)
    top = float(x.max()) if x.numel() else -float("inf")
    if top == -float("inf"):
        return -1, -float("inf"), 1.0
    if u is None or not t > 0:
        return int((x == top).nonzero()[0, 0]), 0.0, 1.0
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    if top == float("inf"):
        w = (x == top).double()
    else:
        w = torch.exp((x - top) / t)
    order = torch.argsort(torch.where(x == 0, 0.0, x), descending=True, stable=True)
    order = order[torch.isfinite(x[order]) | (x[order] == float("inf"))]
    margin = 1.0
    if 0 < k < x.numel():
        order = order[:k]
    if p < 1:
        before = torch.cumsum(w[order], 0) - w[order]
        whole = float(w[order].sum())
        keep = before < p * whole
        keep[0] = True
        off = (before - p * whole).abs()[1:]
        if off.numel():
            margin = min(margin, float(off.min()) / whole)
        order = order[keep]
    if m > 0:
        m = min(m, 1.0)
        off = (w[order] - m).abs()
        margin = min(margin, float(off[off > 0].min()) if (off > 0).any() else 1.0)
        order = order[w[order] >= m]
    order = order.sort().values
    c = torch.cumsum(w[order], 0)
    whole = float(c[-1])
    off = (c[:-1] - u * whole).abs()
    if off.numel():
        margin = min(margin, float(off.min()) / whole)
    n = min(int((c <= u * whole).sum()), order.numel() - 1)
    return int(order[n]), math.log(float(w[order[n]]) / whole) if w[order[n]] > 0 else -float("inf"), margin

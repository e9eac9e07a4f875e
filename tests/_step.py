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

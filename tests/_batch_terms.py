"""Inputs of the batch operators whose results show each term that an F32 value
is kept in, and bounds from the roundings that the kernels state: one product a
sum, so that nothing is added up but a value's own terms.  U is a rounding of
F32 that may cut off, 2^-23; a rounding to nearest is half of it."""
from __future__ import annotations

import torch

U = 2.0 ** -23


def full(shape, g, device, lo=-3, hi=3):
    """F32 values of 24 bits, either sign, magnitudes 2^lo to 2^hi."""
    bits = torch.randint(2 ** 23, 2 ** 24, shape, device=device, generator=g).double()
    e = torch.randint(lo, hi, shape, device=device, generator=g).double()
    sign = torch.randint(0, 2, shape, device=device, generator=g).double() * 2 - 1
    return (sign * bits * 2.0 ** -23 * torch.exp2(e)).float()


# ------------------------------------------------------- low-rank adapters ----
def lora_inputs(device, N, K, M, r, A, dtype, seed):
    """x has one value a token and b one rank an output: a result is the single
    product scale b a x.  (a, b, x, ids, base, scale, result in 64 bits, bound)

    A product of two values: F16's dropped terms (2^-8 of the adapter's value
    times 2^-16 of the activation's) 2^-24, five sums of terms no larger than
    1.01 times the result; twice, and the product with scale.  The terms
    themselves are exact: three BF16 values hold 24 bits.  The base: one rounding.
    A zero may be read for any other product, and sums of zeros are exact."""
    g = torch.Generator(device=device).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    ids = torch.randint(0, A, (N,), device=device, generator=g)
    at = torch.randint(0, K, (N,), device=device, generator=g)
    value = full((N,), g, device)
    x = torch.zeros(N, K, device=device)
    n, m = torch.arange(N, device=device), torch.arange(M, device=device)
    x[n, at] = value
    a = rnd(A, r, K).to(dtype)
    b = torch.zeros(A, M, r, device=device, dtype=dtype)
    b[:, m, m % r] = rnd(A, M).to(dtype)
    scale = full((A,), g, device, -1, 1)
    base = rnd(N, M) * 1e-3
    h = value.double()[:, None] * a[ids, :, at].double()                                   # [N, r]
    term = scale.double()[ids][:, None] * h[:, m % r] * b[:, m, m % r].double()[ids]       # [N, M]
    want = term + base.double()
    return a, b, x, ids.int(), base, scale, want, 12 * U * term.abs() + U * want.abs() + 1e-30


# -------------------------------------------------- shared-prefix attention ----
def score_inputs(device, B, H, hk, D, kv, seed):
    """One key and one dimension a query: the log-sum-exp is the score.
    (q, k, v, lse, bound): two F16 terms leave 2^-22 of the query, the sum of the
    terms, the factor log2 e, the reference and its difference round 8 times
    together; exp2 and log2 are off by units of 7, the exponent of one term."""
    g = torch.Generator(device=device).manual_seed(seed)
    at = torch.randint(0, D, (B, H), device=device, generator=g)
    value = full((B, H), g, device, 3, 6)
    q = torch.zeros(B, H, D, device=device).scatter_(2, at[:, :, None], value[:, :, None])
    k = torch.randn(1, hk, D, device=device, generator=g).to(kv)
    v = torch.randn(1, hk, D, device=device, generator=g).to(kv)
    key = k[0].double().repeat_interleave(H // hk, 0).expand(B, H, D).gather(2, at[:, :, None])[:, :, 0]
    want = value.double() * key
    return q, k, v, want, 10 * U * want.abs() + 2.0 ** -18


def probability_inputs(device, B, H, hk, D, n, kv, seed):
    """One dimension a query and one position a dimension of the values, with n
    <= 64 scores of up to 1.5 (log2): a result is a single probability times a
    value.  (q, k, v, result, bound), the bound in units of U times the result:
    exponents 26 (their terms, references and differences, in the probability and
    in the sum), exp2 4, two F16 terms of a probability 2, their sum 3, the join of
    waves 9, the sum over positions 11, the quotient 3."""
    g = torch.Generator(device=device).manual_seed(seed)
    at = torch.randint(0, D, (B, H), device=device, generator=g)
    value = full((B, H), g, device, -2, -1)
    q = torch.zeros(B, H, D, device=device).scatter_(2, at[:, :, None], value[:, :, None])
    k = torch.randn(n, hk, D, device=device, generator=g).clamp(-2, 2).to(kv)
    d = torch.arange(D, device=device)
    v = torch.zeros(n, hk, D, device=device, dtype=kv)
    v[d % n, :, d] = torch.randn(D, hk, device=device, generator=g).to(kv)
    kd, vd = (t.double().repeat_interleave(H // hk, 1) for t in (k, v))                    # [n, H, D]
    s = value.double()[:, :, None] * kd.permute(1, 2, 0)[None].expand(B, H, D, n).gather(
        2, at[:, :, None, None].expand(B, H, 1, n))[:, :, 0]                               # [B, H, n]
    p = torch.softmax(s, 2)
    want = p[:, :, d % n] * vd[d % n, :, d].t()[None]
    return q, k, v, want, 60 * U * want.abs() + 1e-30

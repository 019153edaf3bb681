"""Attention, its gradients and the key-value cache in 64 bits, with bounds on
what the kernels' roundings can make of a result.

The kernels round the weights P to bf16 as operands (2^-8 of each at most), dS
of d_k to bf16 and of d_q to two bf16 parts, and every result once.  So
  |out - O|  <= 2^-8 (sum P |v| + |O|)
  |d_v - DV| <= 2^-8 (sum P |d_out| + |DV|)
  |d_k - DK| <= 2^-8 (scale sum |dS| |q| + |DK|)
and d_q, whose delta = sum(d_out out) is made of the rounded out: with e the sum of
|d_out| times the bound of out, dS is off by P e, and
  |d_q - DQ| <= scale e sum P |k| + 2^-8 |DQ| + 2^-16 scale sum |dS| |k|.
What FP32 sums and exponentials add is counted as 2^-16 of the sums of magnitudes
that they are made of: 2^-24 a step, some of exp2's argument (below 100), and the
difference dP - delta, whose terms are sums of |d_out| |v| over the columns."""

from __future__ import annotations

import math

HALF = 2.0**-8  # half a step of bf16, relative
FP32 = 2.0**-16


def lengths_of(offsets):
    return [(a, b) for a, b in zip(offsets[:-1], offsets[1:])]


def seen_pairs(n, m, causal, device):
    import torch

    seen = torch.ones(n, m, dtype=torch.bool, device=device)
    return seen.tril(m - n) if causal else seen


def attention64(q, k, v, offsets, key_offsets, causal, scale=None, d_out=None):
    """{name: (result, bound)} in 64 bits; rows of no sequence are 0."""
    import torch

    scale = q.shape[2] ** -0.5 if scale is None else scale
    d = lambda t: t.detach().double()
    q, k, v = d(q), d(k), d(v)
    group = q.shape[1] // k.shape[1]
    zeros = {"out": q, "d_q": q, "d_k": k, "d_v": k}
    got = {n: (torch.zeros_like(t), torch.zeros_like(t)) for n, t in zeros.items()}
    for (a, b), (c, e) in zip(lengths_of(offsets), lengths_of(key_offsets)):
        if a == b:
            continue
        seen = seen_pairs(b - a, e - c, causal, q.device)
        for h in range(q.shape[1]):
            j = h // group
            qq, kk, vv = q[a:b, h], k[c:e, j], v[c:e, j]
            s = (scale * (qq @ kk.t())).masked_fill(~seen, -math.inf)
            top = s.amax(1, keepdim=True) if e > c else s.new_zeros(b - a, 1)
            p = torch.exp(s - top.masked_fill(top == -math.inf, 0))
            total = p.sum(1, keepdim=True)
            p = p / total.masked_fill(total == 0, 1)
            o, spread = p @ vv, p @ vv.abs()
            off = HALF * (spread + o.abs()) + FP32 * spread
            got["out"][0][a:b, h], got["out"][1][a:b, h] = o, off
            if d_out is None:
                continue
            g = d(d_out)[a:b, h]
            dp, dpm = g @ vv.t(), g.abs() @ vv.abs().t()
            delta = (p * dp).sum(1, keepdim=True)
            ds = p * (dp - delta)
            dsm = p * (dpm + (p * dpm).sum(1, keepdim=True))
            worse = (g.abs() * off).sum(1, keepdim=True)
            dq = scale * (ds @ kk)
            got["d_q"][0][a:b, h] = dq
            got["d_q"][1][a:b, h] = (scale * worse * (p @ kk.abs()) + HALF * dq.abs()
                                     + scale * 2 * FP32 * (dsm @ kk.abs()))
            got["d_k"][0][c:e, j] += scale * (ds.t() @ qq)
            got["d_k"][1][c:e, j] += scale * ((HALF * ds.abs() + 2 * FP32 * dsm).t() @ qq.abs())
            got["d_v"][0][c:e, j] += p.t() @ g
            got["d_v"][1][c:e, j] += (HALF + FP32) * (p.t() @ g.abs())
    for name in ("d_k", "d_v"):
        got[name][1].add_(HALF * got[name][0].abs())
    return got


def check(got, want, what=""):
    """Every element of `got` within its bound of the 64-bit result."""
    value, bound = want
    off = (got.detach().double() - value).abs()
    assert bool(got.isfinite().all()), f"{what}: not finite"
    # results of a few 2^-133 are stored as bf16's smallest numbers, whose steps are 2^-133
    over = off - bound * 1.02 - 2.0**-133
    assert bool((over <= 0).all()), f"{what}: off by {float(off.max())}, {float((off / bound.clamp(min=1e-300)).max())} of the bound"


def power(e):
    """2^e in 64 bits by its exponent's bits: a power function's may be off by one step."""
    import torch

    return (e.long() + 1023 << 52).view(torch.float64)


def stored(x, quantised):
    """What a cache holds of rows x [..., dim]: in 64 bits, finite x."""
    import torch

    x = x.double()
    if not quantised:
        return x
    part, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))  # top = part * 2^exponent, part in [0.5, 1)
    e = (exponent - 9 + (part > 0.875)).clamp(min=-117).masked_fill(part == 0, -117)
    y = x * power(-e)
    y = torch.where(e == 120, y.clamp(-240, 240), y)  # the next code would be 2^128
    spacing = power(torch.frexp(y.abs().clamp(min=2.0**-6))[1] - 4)
    return torch.round(y / spacing) * spacing * power(e)

"""Norms and rotation of queries and keys in 64 bits, from the formulas, and how far
fp32 arithmetic with one rounding at the end can be from them.

For a head of D columns x: r = (mean x^2 + eps)^(-1/2).  Every term of a sum of D
squares is off by at most (D + 2) half ulps of the whole (signs of one kind, so
relative): r by (D / 2 + 3) e, e = 2^-24 (the root halves it).  y = x r w: 2 e more;
a turned element is a sum of two products of (y, cos or sin), each off by 2 e more, of
magnitude at most |y_i| + |y_j|.  Backward: g = dy turned back (3 e of |dy_i| + |dy_j|),
dw = sum g u; du = g w; dx = r (du - u m), m = mean(du u) off by (D + 8) e of mean|du u|."""

from __future__ import annotations

import torch

E = 2.0 ** -24
ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-40, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24}


def columns(half, dim, interleaved):
    """the columns of the first and the second of each pair"""
    i = torch.arange(half)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + half)


def turn(y, cos, sin, interleaved, back=False):
    first, second = columns(cos.shape[-1], y.shape[-1], interleaved)
    out = y.clone()
    s = -sin if back else sin
    out[..., first] = y[..., first] * cos - y[..., second] * s
    out[..., second] = y[..., second] * cos + y[..., first] * s
    return out


def spread(y, cos, sin, interleaved):
    """turn()'s sum of magnitudes"""
    first, second = columns(cos.shape[-1], y.shape[-1], interleaved)
    out = y.abs()
    a, b = y[..., first].abs(), y[..., second].abs()
    out[..., first] = a * cos.abs() + b * sin.abs()
    out[..., second] = b * cos.abs() + a * sin.abs()
    return out


def reference(x, w, cos, sin, positions, dy, eps, interleaved):
    """{name: (value, bound)} for x (batch, tokens, heads, dim); cos and sin are the
    float32 tables, which are inputs."""
    dt, dim = x.dtype, x.shape[-1]
    weight = torch.ones(dim, device=x.device) if w is None else w
    wt = weight.dtype
    c, s = (t.double()[positions][..., None, :] for t in (cos, sin))
    x, wd, dy = x.double(), weight.double(), dy.double()
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    er = (dim / 2 + 4) * E
    u = x * r
    y = u * wd
    out = turn(y, c, s, interleaved)
    bound = (er + 6 * E) * spread(y, c, s, interleaved)
    res = dict(y=(out, bound + ULP[dt] * (out.abs() + bound) + TINY[dt]))

    g = turn(dy, c, s, interleaved, back=True)
    eg = 3 * E * spread(dy, c, s, interleaved)
    du = g * wd
    edu = eg * wd.abs() + E * du.abs()
    m = (du * u).mean(-1, keepdim=True)
    em = (edu * u.abs()).mean(-1, keepdim=True) + (dim + 8 + dim / 2 + 4) * E * (
        du * u).abs().mean(-1, keepdim=True)
    dx = r * (du - u * m)
    edx = r * (edu + u.abs() * em) + (er + 4 * E) * r * (du.abs() + (u * m).abs())
    res["dx"] = (dx, edx + ULP[dt] * (dx.abs() + edx) + TINY[dt])
    if w is not None:
        n = x.shape[0] * x.shape[1] * x.shape[2]
        dw = (g * u).sum((0, 1, 2))
        # sums of n terms in any order: n roundings of a partial sum at worst
        edw = (eg * u.abs() + (er + (min(n, 4096) + 8) * E) * (g * u).abs()).sum((0, 1, 2))
        res["dw"] = (dw, edw + ULP[wt] * (dw.abs() + edw) + TINY[wt])
    return res

"""The gated feed-forward block in 64 bits, and how far a result that rounds
where the kernels say they round can be from it.

Bounds are elementwise and propagate worst cases: a sum of K products in fp32
is off by at most (K + 8) 2^-24 times the sum of the products' magnitudes (for
fp32 inputs 2^-22 of it more: the dropped parts of split products); h, da and
db are rounded to the type (half an ulp, u); a and b are kept with 16
significant bits for 16-bit types; f and f' are good to 1e-6 of their largest
factor; f'' is at most 1.2 in magnitude for every f (relu's jump is allowed for
where a's error reaches zero)."""

from __future__ import annotations

import math

import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# spacing of the subnormal numbers
TINY = {torch.float32: 1e-40, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24}


def act(name, a):
    """f(a) and f'(a)"""
    if name in ("silu", "sigmoid"):
        s = torch.sigmoid(a)
        return (a * s, s * (1 + a * (1 - s))) if name == "silu" else (s, s * (1 - s))
    if name == "relu":
        on = (a > 0).to(a.dtype)
        return a * on, on
    if name == "gelu":
        c = 0.5 * torch.erfc(-a * math.sqrt(0.5))
        return a * c, c + a * torch.exp(-0.5 * a * a) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (a + 0.044715 * a ** 3))
    return (0.5 * a * (1 + t),
            0.5 * (1 + t) + 0.5 * a * (1 - t * t) * k * (1 + 3 * 0.044715 * a * a))


def reference(x, wg, wu, wd, dy, name):
    """{output: (value, bound)} in float64 for 2-D inputs of the type under test."""
    dt = x.dtype
    u, tiny = U[dt], TINY[dt]
    extra = 2.0 ** -22 if dt == torch.float32 else 0.0
    kept = 2.0 ** -15 if dt != torch.float32 else 0.0
    x, wg, wu, wd, dy = (t.detach().double() for t in (x, wg, wu, wd, dy))
    (tokens, d), f = x.shape, wg.shape[0]

    def product(a, b, ea=None, eb=None):
        """a b^T, its bound from the factors' errors and its own sum's"""
        k = a.shape[1]
        mag = a.abs() @ b.abs().t()
        err = mag * ((k + 8) * 2.0 ** -24 + extra)
        if ea is not None:
            err = err + ea @ b.abs().t()
        if eb is not None:
            err = err + a.abs() @ eb.t()
        return a @ b.t(), err

    a, ea = product(x, wg)
    b, eb = product(x, wu)
    fa, ga = act(name, a)
    h = fa * b
    fmag, efa = a.abs() + 1, ga.abs() * ea + 1.2 * ea * ea
    eh = efa * (b.abs() + eb) + fa.abs() * eb + 1e-6 * fmag * b.abs()
    eh = eh + u * (h.abs() + eh) + tiny
    y, ey = product(h, wd, eh)
    out = dict(y=(y, ey))

    dh, edh = product(dy, wd.t())
    ea2, eb2 = ea + kept * a.abs(), eb + kept * b.abs()
    ega = 1.2 * ea2 + 2e-6 * fmag
    if name == "relu":
        ega = (a.abs() <= ea2).double()
    da, db = dh * b * ga, dh * fa
    eda = (edh * (b.abs() + eb2) * (ga.abs() + ega) + dh.abs() * eb2 * (ga.abs() + ega)
           + (dh * b).abs() * ega) * (1 + 1e-6) + da.abs() * 3e-7
    efa2 = ga.abs() * ea2 + 1.2 * ea2 * ea2 + 1e-6 * fmag
    edb = edh * (fa.abs() + efa2) + dh.abs() * efa2 + db.abs() * 2e-7
    eda, edb = (e + u * (v.abs() + e) + tiny for v, e in ((da, eda), (db, edb)))
    x1, e1 = product(da, wg.t(), eda)
    x2, e2 = product(db, wu.t(), edb)
    out["dx"] = (x1 + x2, e1 + e2 + f * 2.0 ** -24 * (da.abs() @ wg.abs() + db.abs() @ wu.abs()))
    out["dgate"] = product(da.t(), x.t(), eda.t())
    out["dup"] = product(db.t(), x.t(), edb.t())
    out["ddown"] = product(dy.t(), h.t(), None, eh.t())
    return {k: (v, e + u * (v.abs() + e) + tiny) for k, (v, e) in out.items()}


def norm_bound(dtype):
    """Largest relative error of a whole output in the 2-norm: a rounding to the
    type is at most u an element and, spread evenly, u / sqrt 3; an output
    passes at most four of them (its own, and those of two factors and h): 2 u.
    fp32's sums of up to 30000 products of random signs: 1e-5."""
    return 2 * U[dtype] if dtype != torch.float32 else 1e-5

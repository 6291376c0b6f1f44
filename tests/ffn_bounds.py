"""How far a whole output of the feed-forward block may be from its definition in
the 2-norm, from the sizes of its roundings: narrow enough to tell a lost part.

fp32 (units of 2^-24, u).  A product of K terms rounds at most once a term, by
u / sqrt 3 of the partial sum on average, in the last of its six segments (the
others' sums are 2^-8 of it and less); partial sums of terms of random signs
grow as the square root, half the last one's square on average; joining parts
rounds up to 32 times more, and the dropped parts of the operands are 2^-26.  So
e(K) = 3 + 0.41 sqrt K.  An activation is good to 4 u, and none of the five
enlarges its argument's error in the norm.  Errors of different roundings are
independent and add up as squares:

  y      e(f), and h's: two projections e(d), an activation
  dx     e(2 f), and da's and db's: dh, a and b e(d), an activation
  dgate  e(tokens), and da's, ...

16-bit types (units of u, half an ulp at 1: 2^-8, 2^-11).  Evenly spread over a
binade, a rounding is 0.42 u of what is rounded; every output passes two, its own
and that of the factor h, da or db: 0.59 u.  Half as much again is not reached."""

from __future__ import annotations

import math

import torch

from tests.ffn_reference import U

OUTPUTS = ("y", "dx", "dgate", "dup", "ddown")


def norm_bound(dtype, output, tokens, d, f):
    u = U[dtype]
    if dtype != torch.float32:
        return 0.8 * u
    e = lambda k: 3 + 0.41 * math.sqrt(k)   # noqa: E731
    own = e({"y": f, "dx": 2 * f}.get(output, tokens))
    return u * math.sqrt(own ** 2 + (2 if output in ("y", "ddown") else 3) * e(d) ** 2 + 2 * 4 ** 2)

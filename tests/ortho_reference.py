"""Newton-Schulz orthogonalisation in 64 bits, and how far a result that rounds
where the kernels say they round can be from it, in the Frobenius norm.

A step is the odd matrix function p(s) = a s + b s^3 + c s^5 of the singular
values; in the Frobenius norm it enlarges an error by at most the largest
|p'(s)| on the singular values' range (the divided differences of an odd
function on [-u, u] are values of its derivative).  Its own errors:

  words: X, A and B are rounded to words, relative w an element: 2^-11 (fp16) or,
    with two words, 2^-22 (of which the lower word's rounding is one half, the
    dropped product of two lower words the other);
  sums: a sum of K products in fp32 rounds K times by half an ulp of a partial
    sum, signs at random: sqrt(K) 2^-24 of the product of the factors' norms,
    and four times that for what a partial sum may exceed its end.

Errors of A reach B as |b| + 2 |c| |A|, errors of B reach X times |X|, both in the
spectral norm.

Matrices of up to 512 x 1024 may take their steps by panels: Y = A X, A'' = Y X^T and
Z = A'' X instead of A A and B X, a X + b Y + c Z in fp32.  An error of A reaches Y times
|X|, one of Y reaches A'' times |X|, one of A'' reaches Z times |X|; Y and A'' are
rounded to words where they are a product's factor (b Y is not), and every product has
the sums' and the dropped words' errors.  The larger of the two ways' errors counts."""

from __future__ import annotations

import math

import torch

WORD = {"fast": 2.0 ** -11, "fp32": 2.0 ** -22}
ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
CUBIC, QUINTIC = (1.5, -0.5, 0.0), (1.875, -1.25, 0.375)


def orthogonalize(g, coefficients, eps=1e-7):
    """One matrix in float64; coefficients: a triple for every step."""
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.square().sum().sqrt() + eps)
    for a, b, c in coefficients:
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if tall else x


def _sums(k):
    return 4 * math.sqrt(k) * 2.0 ** -24


def bound(g, coefficients, precision, eps=1e-7):
    """Largest error of the result in the Frobenius norm (absolute), before it is
    rounded to its type."""
    w = WORD[precision]
    x = g.double()
    x = x.t() if x.shape[0] > x.shape[1] else x
    s, l = x.shape
    x = x / (x.square().sum().sqrt() + eps)
    u, err = 1.0, 2 * w * float(x.norm())
    for a, b, c in coefficients:
        grid = torch.linspace(0, u, 4001, dtype=torch.float64)
        slope = float((a + 3 * b * grid ** 2 + 5 * c * grid ** 4).abs().max())
        gram = x @ x.t()
        top = float(torch.linalg.matrix_norm(gram, 2)) + 1e-30   # |A| in the spectral norm
        square = gram @ gram
        factor = b * gram + c * square
        nx, na = float(x.norm()), float(gram.norm())
        ea = w * na + _sums(l) * nx * nx + 2 * w * math.sqrt(top) * nx
        eb = (abs(b) + 2 * abs(c) * top) * ea + w * float(factor.norm()) + (
            _sums(s) + 2 * w) * abs(c) * na * na
        ex = math.sqrt(top) * eb + (_sums(s) + 2 * w) * float(
            factor.norm()) * nx + 2.0 ** -23 * abs(a) * nx
        if s <= 512 and l <= 1024:
            y, z = gram @ x, square @ x
            ny, nz, root = float(y.norm()), float(z.norm()), math.sqrt(top)
            ey = root * ea + (_sums(s) + 2 * w) * na * nx
            e2 = root * (ey + w * ny) + (_sums(l) + 2 * w) * ny * nx + w * float(square.norm())
            ez = root * e2 + (_sums(s) + 2 * w) * float(square.norm()) * nx
            ex = max(ex, abs(b) * ey + abs(c) * ez
                     + 2.0 ** -22 * (abs(a) * nx + abs(b) * ny + abs(c) * nz))
        x = a * x + factor @ x
        err = slope * err + ex + w * float(x.norm())
        u = float((a * grid + b * grid ** 3 + c * grid ** 5).abs().max())
    return err


def triples(coefficients, steps):
    return [tuple(coefficients)] * steps

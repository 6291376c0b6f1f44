"""How far orthogonalised updates of one word an element may be from the definition: as
far as products whose factors are rounded to 11 significant bits once a step, and no
further.

``emulate`` takes the steps in 64 bits and rounds X, A and B, and those alone, to 11 bits
where the next product takes them.  Its error is a sum of some 3 roundings a step of tens
of thousands of elements each, independent of one another, so that their squares add up:
another set of roundings of the same sizes (sums in another order, the same matrix under
another seed) gives the same Frobenius norm to within a few hundredths.  The result's own
rounding, which is computed from the exact result, adds its square.  ``allowed`` is that
sum's root and 15% for what the few strong singular values, whose errors are few numbers
and not thousands, may differ by.  A word of ten bits instead of eleven would double the
first part, which is the larger one where the result is float32, and 0.6 of the second
where it is bfloat16: 1.6 times the root."""

from __future__ import annotations

import torch

from tests.ortho_reference import orthogonalize, triples

PUBLISHED = triples((3.4445, -4.7750, 2.0315), 5)


def rounded(m, bits=11):
    mantissa, exponent = torch.frexp(m)
    return torch.ldexp(torch.round(mantissa * 2.0 ** bits) / 2.0 ** bits, exponent)


def emulate(g, coefficients, bits=11, eps=1e-7):
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = rounded(x / (x.square().sum().sqrt() + eps), bits)
    eye = torch.eye(x.shape[0], dtype=x.dtype, device=x.device)
    for k, (a, b, c) in enumerate(coefficients):
        gram = rounded(x @ x.t(), bits)
        x = rounded(a * eye + b * gram + c * (gram @ gram), bits) @ x
        if k + 1 < len(coefficients):
            x = rounded(x, bits)
    return x.t() if tall else x


def relative(got, want):
    return float((got.double() - want).norm() / want.norm())


def allowed(g, coefficients, dtype, bits=11):
    """the exact result, and the relative error that one in dtype may have"""
    want = orthogonalize(g, coefficients)
    words = relative(emulate(g, coefficients, bits), want)
    own = relative(want.to(dtype), want)
    return want, 1.15 * (words ** 2 + own ** 2) ** 0.5

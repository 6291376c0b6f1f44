"""That the bounds of tests/ortho_words.py tell one scheme of roundings from another."""

from __future__ import annotations

import pytest
import torch

from tests.ortho_reference import orthogonalize
from tests.ortho_words import PUBLISHED, allowed, emulate, relative, rounded


def _update(m, n, seed=0):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(m, n, generator=g)
    t += torch.randn(m, 2, generator=g) @ torch.randn(2, n, generator=g) * ((m + n) / (m * n)) ** 0.5
    return (t * 1e-3).bfloat16()


def _panels(g, inner):
    """panels of A and A A of `inner` bits, X and A X of 11"""
    x = g.double()
    x = rounded(x / x.norm())
    for k, (a, b, c) in enumerate(PUBLISHED):
        gram = rounded(x @ x.t(), inner)
        y = gram @ x
        square = rounded(rounded(y) @ x.t(), inner)
        x = a * x + b * y + c * (square @ x)
        x = rounded(x) if k + 1 < len(PUBLISHED) else x
    return x


@pytest.mark.parametrize("m,n", [(160, 160), (256, 256), (256, 1024), (200, 300)])
def test_what_the_bounds_let_through(m, n):
    g = _update(m, n)
    for dtype in (torch.float32, torch.bfloat16):
        want, room = allowed(g, PUBLISHED, dtype)
        assert room <= 2.7e-3   # in bfloat16; in float32 the words alone, 1.4e-3, and 15%
        assert dtype != torch.float32 or room <= 1.62e-3
        # other data of the same kind, and panels with A in 22 bits
        twin = _update(m, n, 1)
        other = relative(emulate(twin, PUBLISHED).to(dtype), orthogonalize(twin, PUBLISHED))
        assert other <= room
        assert relative(_panels(g, 22).to(dtype), want) <= room
        # not a word of ten bits; not panels all of whose words have eleven; not the
        # update of one step less, or one of the others
        assert relative(emulate(g, PUBLISHED, 10).to(dtype), want) > room
        if dtype == torch.float32 or n >= 1024:
            assert relative(_panels(g, 11).to(dtype), want) > room
        assert relative(orthogonalize(g, PUBLISHED[:4]).to(dtype), want) > 10 * room
        assert relative(torch.zeros_like(want), want) > 100 * room


def test_rounding():
    x = torch.tensor([1.0, 1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 0.0, -3.0, 2049.0],
                     dtype=torch.float64)
    assert torch.equal(rounded(x), x.half().double())

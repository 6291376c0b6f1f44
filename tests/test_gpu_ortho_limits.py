"""The orthogonalised updates at the ends of what is allowed: longest sides, more than 2^31
elements, most steps."""

from __future__ import annotations

import pytest
import torch

import scao_amd
from scao_amd import _lib as L
from tests.ortho_reference import QUINTIC, ULP, bound, orthogonalize, triples
from tests.test_gpu_ortho import _update

pytestmark = pytest.mark.gpu

LONGEST = (1 << 20) - 1


@pytest.mark.parametrize("m,n,dtype", [(1, LONGEST, torch.float32), (LONGEST, 1, torch.bfloat16),
                                       (2, LONGEST, torch.float16), (LONGEST, 3, torch.float32),
                                       (130, LONGEST, torch.float32),
                                       (LONGEST, 131, torch.bfloat16)])
def test_longest_sides(hip_device, m, n, dtype):
    g = _update(hip_device, 2, m, n, dtype)
    precision = "fast" if dtype == torch.bfloat16 else "fp32"
    got = scao_amd.orthogonalize(g, steps=2, coefficients=QUINTIC)
    want = orthogonalize(g, triples(QUINTIC, 2))
    room = bound(g, triples(QUINTIC, 2), precision) + ULP[dtype] * float(want.norm())
    err = float((got.double() - want).norm())
    print(f"{m}x{n}: {err:.2e} of {room:.2e}", flush=True)
    assert err <= room < 0.05 * float(want.norm())


def _ones(dev, s, l, tall, dtype):
    """one 1 in every row (of the smaller side), no two in a column; and where they are"""
    g = torch.Generator(device=dev).manual_seed(1)
    at = torch.randperm(l, generator=g, device=dev)[:s]
    t = torch.zeros((l, s) if tall else (s, l), device=dev, dtype=dtype)
    i = torch.arange(s, device=dev)
    index = (at, i) if tall else (i, at)
    t[index] = 1
    return t, index


@pytest.mark.parametrize("tall", [False, True])
def test_past_2_to_the_31_elements(hip_device, tall):
    """X = 2^-7 at the ones, A = 2^-14 on the diagonal, B = 1.5 - 2^-15 there, of which
    words of 11 bits keep 1.5, and X <- B X: whatever lies elsewhere stays zero."""
    s, l = 1 << 14, (1 << 17) + 8
    g, index = _ones(hip_device, s, l, tall, torch.bfloat16)
    assert g.numel() > 1 << 31
    got = scao_amd.orthogonalize(g, steps=1, coefficients=(1.5, -0.5, 0.0), eps=1e-30)
    assert bool((got[index] == 1.5 / 128).all())
    assert int(torch.count_nonzero(got)) == s
    # a step of Muon: p <- 0.5 p - 64 O
    del got
    p = torch.zeros_like(g)
    p[-1, -1] = 2.0
    last = bool(g[-1, -1] == 1)
    momentum = torch.zeros(g.shape, device=hip_device)
    L.torch_host().muon_step([p], [g], [momentum], [64.0], [0.5], 0.5, False, [1.5, -0.5, 0.0],
                             1e-30, [L.ORTHO_FAST])
    assert float(p[-1, -1]) == (1.0 - 0.75 if last else 1.0)
    p[-1, -1] = 0
    inside = (index[0] != g.shape[0] - 1) | (index[1] != g.shape[1] - 1)
    assert bool((p[index][inside] == -0.75).all())
    assert int(torch.count_nonzero(p)) == int(inside.sum())
    assert int(torch.count_nonzero(momentum)) == s and bool((momentum[index] == 0.5).all())


@pytest.mark.parametrize("steps", [16, 17, 64])
@pytest.mark.parametrize("m,n", [(40, 64), (128, 100), (300, 200), (700, 530)])
def test_many_steps(hip_device, m, n, steps):
    """Singular values that start at 1 / sqrt(n), up to a factor of 4, are all 1 after a
    dozen quintic steps: the polar factor.  Later steps turn it by their roundings, at most
    four of 2^-22 each beside sums' and the start's (6e-6 for all of them)."""
    g = torch.Generator().manual_seed(m)
    u, _, v = torch.linalg.svd(torch.randn(m, n, generator=g, dtype=torch.float64),
                               full_matrices=False)
    x = (u * torch.logspace(0, 0.6, min(m, n), dtype=torch.float64)) @ v
    got = scao_amd.orthogonalize(x.float().to(hip_device), steps=steps, coefficients=QUINTIC)
    err = float((got.cpu().double() - u @ v).norm() / min(m, n) ** 0.5)
    print(f"{m}x{n}, {steps} steps: {err:.2e}", flush=True)
    assert err <= 4 * steps * 2.0 ** -22 + 6e-6

"""Gradient norm and clipping at the ends of what they take: gradients that
only an iterator holds, versions, bounds of infinity, shared memory, tracing.

The norm of small whole numbers is exact; scaled values are compared with the
product in 64 bits, rounded once."""

from __future__ import annotations

import math

import pytest
import torch

import scao_amd

pytestmark = pytest.mark.gpu


def _params(grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype, device=g.device))
        p.grad = g
        out.append(p)
    return out


def _normal(dev, seed, *shape, dtype=torch.float32, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(dev)


def test_gradients_that_only_an_iterator_holds(hip_device):
    """They live until the kernels are queued: in several tables, the memory of
    the last ones freed first would hold the first table's sums."""
    torch.cuda.empty_cache()
    for entry in (scao_amd.global_grad_norm, lambda p: scao_amd.clip_grad_norm_(p, 1.0)):
        params = _params([torch.ones(4000, device=hip_device) for _ in range(1000)])

        def temporaries():
            while params:
                yield params.pop()

        torch.cuda.synchronize()
        assert entry(temporaries()).item() == 2000.0

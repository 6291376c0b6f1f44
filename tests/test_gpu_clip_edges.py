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


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_a_bound_of_infinity_clips_nothing(hip_device, p, scale):
    """max_norm = inf measures: the factor is `scale`, with an infinite norm too."""
    for bad in (None, math.inf, -math.inf):
        g, h = _normal(hip_device, 4, 20000), _normal(hip_device, 5, 7, dtype=torch.bfloat16)
        if bad is not None:
            g[12345] = bad
        want = [t * scale for t in (g, h)]
        norm = scao_amd.clip_grad_norm_(_params([g, h]), math.inf, norm_type=p, scale=scale)
        assert norm.item() == math.inf if bad is not None else math.isfinite(norm.item())
        assert torch.equal(g, want[0]) and torch.equal(h, want[1])
    g[3] = math.nan
    norm = scao_amd.clip_grad_norm_(_params([g, h]), math.inf, norm_type=p)
    assert math.isnan(norm.item()) and bool(g.isnan().all()) and bool(h.isnan().all())

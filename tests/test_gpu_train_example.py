"""The example that runs the feed-forward block, the clipping and SCAO together."""

from __future__ import annotations

import importlib.util
import math
import os

import pytest
import torch

import scao_amd

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location(
        "train_ffn", os.path.join(ROOT, "examples", "train_ffn.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_it_learns(hip_device, dtype):
    history = _example().train(steps=60, dtype=dtype, log=lambda s: print(s, flush=True))
    assert all(math.isfinite(v) for pair in history for v in pair)
    first = sum(v for v, _ in history[:3]) / 3
    last = sum(v for v, _ in history[-3:]) / 3
    assert last < 0.1 * first, (first, last)
    assert history[0][1] > 1.0   # the first steps are clipped


def test_a_step_equals_the_plain_one(hip_device):
    """Gradients of two micro-batches through the block, averaged and clipped,
    against elementary operations in 64 bits on the same weights (fp32; the
    tolerance is the sums' 1e-5)."""
    torch.manual_seed(1)
    model = _example().Stack(2, 64, 96, device=hip_device)
    xs = [torch.randn(30, 64, device=hip_device) for _ in range(2)]

    def plain(params):
        total = None
        for x in xs:
            h = x.double()
            for block in model.blocks:
                w = {k: params[id(p)] for k, p in block.named_parameters()}
                gate, up = w["gate_up"].split(96) if block.packed else (w["gate"], w["up"])
                h = h + (torch.nn.functional.silu(h @ gate.t()) * (h @ up.t())) @ w["down"].t()
            loss = h.square().mean()
            total = loss if total is None else total + loss
        return total

    wide = {id(p): p.detach().double().requires_grad_() for p in model.parameters()}
    grads = torch.autograd.grad(plain(wide), list(wide.values()))
    norm = torch.cat([g.reshape(-1) for g in grads]).norm() / 2
    for x in xs:
        model(x).square().mean().backward()
    got = scao_amd.clip_grad_norm_(model.parameters(), 0.01, scale=0.5)
    assert abs(got.item() - norm.item()) <= 1e-5 * norm.item()
    for p, g in zip(model.parameters(), grads):
        want = g * (0.5 * min(1.0, 0.01 / (norm.item() + 1e-6)))
        assert (p.grad.double() - want).norm() <= 2e-5 * want.norm()

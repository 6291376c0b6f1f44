"""examples/train_decoder.py: the operators together, as a training program calls
them.  It runs, its gradients are those of the same model written in elementary
torch operations in 64 bits, and its steps are the optimisers' own."""

from __future__ import annotations

import importlib.util
import math
import os

import pytest
import torch

import scao_amd
from tests.ortho_reference import bound, orthogonalize, triples

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location(
        "train_decoder", os.path.join(ROOT, "examples", "train_decoder.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_it_runs(hip_device, example, dtype):
    lines = []
    history = example.train(steps=4, dtype=dtype, log=lines.append)
    assert len(history) == 4 and len(lines) == 2
    assert all(math.isfinite(x) for pair in history for x in pair)


def _plain(model, w, tokens):
    """The decoder's logits from its parameters w in float64."""
    def rms(x, weight, eps):
        return x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * weight

    def turn(y, cos, sin):
        half = cos.shape[-1]
        a, b = y[..., :half], y[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    x = w["embedding.weight"][tokens]
    eps = torch.finfo(torch.float32).eps   # nn.RMSNorm's default for its inputs
    for i, layer in enumerate(model.layers):
        p = {k[len(f"layers.{i}."):]: v for k, v in w.items() if k.startswith(f"layers.{i}.")}
        h, kv, d, t = layer.heads, layer.kv_heads, layer.dim, tokens.shape[1]
        rows = (rms(x, p["norms.0.weight"], eps) @ p["qkv.weight"].t()).unflatten(-1, (-1, d))
        q, k, v = rows.split([h, kv, kv], -2)
        cos, sin = (s[:t].double()[:, None] for s in (layer.rope.cos, layer.rope.sin))
        q = turn(rms(q, p["rope.q"], 1e-6), cos, sin)
        k = turn(rms(k, p["rope.k"], 1e-6), cos, sin)
        share = torch.arange(h, device=x.device) // (h // kv)
        q, k, v = q.transpose(1, 2), k[:, :, share].transpose(1, 2), v[:, :, share].transpose(1, 2)
        logits = q @ k.mT.contiguous() / math.sqrt(d)
        later = torch.ones(t, t, dtype=torch.bool, device=x.device).triu(1)
        mixed = logits.masked_fill(later, -math.inf).softmax(-1) @ v
        x = x + mixed.transpose(1, 2).flatten(2) @ p["out.weight"].t()
        z = rms(x, p["norms.1.weight"], eps)
        gate, up = (z @ p["ffn.gate_up"].t()).chunk(2, -1)
        x = x + (gate * torch.sigmoid(gate) * up) @ p["ffn.down"].t()
    return rms(x, w["norm.weight"], eps) @ w["embedding.weight"].t()


def _model(example, dev):
    torch.manual_seed(3)
    model = example.Decoder(vocabulary=50, layers=2, d_model=96, heads=6, kv_heads=2, d_ff=136,
                            length=40, device=dev, dtype=torch.float32)
    with torch.no_grad():
        for name, p in model.named_parameters():
            if p.ndim == 1:
                p.copy_(1 + 0.2 * torch.randn_like(p))
    return model, torch.randint(50, (3, 37), device=dev)


def test_gradients(hip_device, example):
    model, tokens = _model(example, hip_device)
    dy = torch.randn(3, 37, 50, device=hip_device) * 0.1
    model(tokens).backward(dy)
    w = {k: v.detach().double().requires_grad_() for k, v in model.named_parameters()}
    _plain(model, w, tokens).backward(dy.double())
    for name, p in model.named_parameters():
        want = w[name].grad
        err = float((p.grad.double() - want).norm() / want.norm())
        # fp32 products and sums of up to 5000 terms, some fifteen of them after one
        # another: 15 sqrt(5000) 2^-24 = 6e-5
        assert err <= 6e-5, (name, err)


def test_a_step_of_both_optimisers(hip_device, example):
    model, tokens = _model(example, hip_device)
    opts = example.optimizers(model, 0.05)
    names = {id(p): n for n, p in model.named_parameters()}
    owned = [[names[id(p)] for p in o.param_groups[0]["params"]] for o in opts]
    assert sorted(owned[0] + owned[1]) == sorted(names.values())
    assert all("layers" in n for n in owned[0]) and "embedding.weight" in owned[1]
    model(tokens).float().square().mean().backward()
    norm = scao_amd.clip_grad_norm_(model.parameters(), 0.5)
    grads = [p.grad.double() for p in model.parameters()]
    total = math.sqrt(sum(float(g.square().sum()) for g in grads))
    assert abs(total - min(0.5, float(norm))) <= 1e-4 * total
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    for o in opts:
        o.step()
    co = triples(scao_amd.ortho.NS_COEFFICIENTS, 5)
    for n, p in model.named_parameters():
        assert bool(p.isfinite().all()) and not torch.equal(p, before[n])
        if n in owned[0]:
            # the first step: m = 0.05 g, u = 0.95 m + 0.05 g
            u = (0.95 * 0.05 + 0.05) * p.grad.double()
            rate = 0.05 * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
            want = (1 - 0.05 * 0.01) * before[n].double() - rate * orthogonalize(u, co)
            room = rate * (bound(u, co, "fp32") + 1e-5 * min(p.shape) ** 0.5) + 3e-7 * float(
                before[n].norm())
            assert float((p.detach().double() - want).norm()) <= room, n

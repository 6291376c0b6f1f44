"""The step of Muon (scao_muon_step) against its definition in 64 bits; the
orthogonalised update's bounds are tests/ortho_reference.py's."""

from __future__ import annotations

import copy
import math

import pytest
import torch

import scao_amd
from tests.ortho_reference import QUINTIC, ULP, bound, orthogonalize, triples

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(96, 160), (160, 96), (50, 333), (64, 64), (1, 40), (33, 1), (3, 40, 72)]


def _model(dev, dtype, seed=0, grad_dtype=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    params = []
    for shape in SHAPES:
        p = torch.nn.Parameter((torch.randn(shape, generator=g, device=dev) * 0.05).to(dtype))
        p.grad = (torch.randn(shape, generator=g, device=dev) * 1e-2).to(dtype)
        params.append(p)
    return params


def _reference(p, grad, buf, lr, wd, mu, nesterov, co, adjust, precision):
    """p, the momentum, and the bound of p's error, of one matrix in float64"""
    g = grad.double()
    buf = mu * buf + (1 - mu) * g
    u = mu * buf + (1 - mu) * g if nesterov else buf
    rows, cols = p.shape
    ratio = (0.2 * math.sqrt(max(rows, cols)) if adjust == "match_rms_adamw"
             else math.sqrt(max(1.0, rows / cols)))
    new = (1 - lr * wd) * p.double() - lr * ratio * orthogonalize(u, co)
    # u itself is off by three roundings of 2^-24, the sum of p by two
    room = lr * ratio * (bound(u, co, precision) + 4e-7 * min(rows, cols) ** 0.5 * 16)
    return new, buf, room + (ULP[p.dtype] + 2.0 ** -22) * float(new.norm() + p.double().norm())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("adjust", [None, "match_rms_adamw"])
def test_steps(hip_device, dtype, nesterov, adjust):
    lr, wd, mu, co = 0.03, 0.2, 0.9, triples(QUINTIC, 2)
    params = _model(hip_device, dtype)
    opt = scao_amd.Muon(params, lr=lr, weight_decay=wd, momentum=mu, nesterov=nesterov,
                        ns_coefficients=QUINTIC, ns_steps=2, adjust_lr_fn=adjust)
    momenta = [torch.zeros(p.shape, dtype=torch.float64, device=hip_device) for p in params]
    precision = "fp32" if dtype == torch.float32 else "fast"
    for step in range(3):
        before = [p.detach().clone() for p in params]
        for i, p in enumerate(params):
            p.grad = torch.randn(p.shape, device=hip_device).mul_(1e-2).to(dtype)
        opt.step()
        for p, old, m in zip(params, before, momenta):
            buf = opt.state[p]["momentum_buffer"]
            assert buf.dtype == torch.float32
            for k in range(p.shape[0] if p.ndim == 3 else 1):
                at = (k,) if p.ndim == 3 else ()
                want, mom, room = _reference(old[at], p.grad[at], m[at], lr, wd, mu, nesterov, co,
                                             adjust, precision)
                err = float((p.detach()[at].double() - want).norm())
                assert err <= room, (step, p.shape, err, room)
                # (two roundings a step of values that the last one's error scales)
                assert torch.allclose(buf[at].double(), mom, rtol=0,
                                      atol=4 * 2.0 ** -24 * (step + 1) * float(mom.abs().max()))
                m[at] = mom


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nesterov", [True, False])
def test_steps_of_a_few_hundred_rows(hip_device, dtype, nesterov):
    lr, wd, mu, co = 0.03, 0.2, 0.9, triples(QUINTIC, 2)
    params = [torch.nn.Parameter((torch.randn(shape, device=hip_device) * 0.05).to(dtype))
              for shape in ((256, 256), (300, 160), (2, 140, 333))]
    opt = scao_amd.Muon(params, lr=lr, weight_decay=wd, momentum=mu, nesterov=nesterov,
                        ns_coefficients=QUINTIC, ns_steps=2)
    momenta = [torch.zeros(p.shape, dtype=torch.float64, device=hip_device) for p in params]
    precision = "fp32" if dtype == torch.float32 else "fast"
    for step in range(2):
        before = [p.detach().clone() for p in params]
        for p in params:
            p.grad = torch.randn(p.shape, device=hip_device).mul_(1e-2).to(dtype)
        opt.step()
        for p, old, m in zip(params, before, momenta):
            for k in range(p.shape[0] if p.ndim == 3 else 1):
                at = (k,) if p.ndim == 3 else ()
                want, mom, room = _reference(old[at], p.grad[at], m[at], lr, wd, mu, nesterov, co,
                                             None, precision)
                err = float((p.detach()[at].double() - want).norm())
                assert err <= room, (step, p.shape, err, room)
                m[at] = mom


@pytest.mark.parametrize("ns_dtype,precision", [(torch.bfloat16, "fast"), (torch.float32, "fp32")])
def test_precision_by_choice(hip_device, ns_dtype, precision):
    for dtype in (torch.float32, torch.bfloat16):
        p = _model(hip_device, dtype)[0]
        old = p.detach().clone()
        scao_amd.Muon([p], lr=0.5, weight_decay=0.0, ns_coefficients=QUINTIC, ns_steps=2,
                      ns_dtype=ns_dtype).step()
        want, _, room = _reference(old, p.grad, 0.0, 0.5, 0.0, 0.95, True, triples(QUINTIC, 2),
                                   None, precision)
        assert float((p.detach().double() - want).norm()) <= room


def test_mixed_groups_and_missing_gradients(hip_device):
    """Groups of their own rates; gradients of another type, strided; a parameter
    without one is left alone."""
    params = _model(hip_device, torch.float32)
    twin = copy.deepcopy(params)
    for p, q in zip(params, twin):
        q.grad = p.grad.clone()
    params[0].grad = None
    twin[0].grad = None
    params[1].grad = params[1].grad.t().contiguous().t()
    opt = scao_amd.Muon([dict(params=params[:3], lr=0.1), dict(params=params[3:], momentum=0.5)])
    one = [scao_amd.Muon([q], lr=0.1 if i < 3 else 1e-3, momentum=0.95 if i < 3 else 0.5)
           for i, q in enumerate(twin)]
    before = params[0].detach().clone()
    versions = [p._version for p in params]
    opt.step()
    for o in one:
        o.step()
    assert torch.equal(params[0], before) and params[0] not in opt.state
    assert [p._version > v for p, v in zip(params, versions)] == [False] + [True] * 6
    for p, q in zip(params[1:], twin[1:]):
        # company may cut a matrix's sums differently
        assert torch.allclose(p, q, rtol=0, atol=1e-5)


def test_state_survives_a_checkpoint(hip_device):
    for dtype in TYPES:
        params, twin = _model(hip_device, dtype), _model(hip_device, dtype)
        a, b = scao_amd.Muon(params, lr=0.02), scao_amd.Muon(twin, lr=0.5)
        a.step()
        for p, q in zip(params, twin):
            q.data.copy_(p.data)
        b.load_state_dict(copy.deepcopy(a.state_dict()))
        for p, q in zip(params, twin):
            assert torch.equal(a.state[p]["momentum_buffer"], b.state[q]["momentum_buffer"])
            assert b.state[q]["momentum_buffer"].dtype == torch.float32
        a.step()
        b.step()
        assert all(torch.equal(p, q) for p, q in zip(params, twin))


def test_a_nan_gradient_stays_in_its_matrix(hip_device):
    params = _model(hip_device, torch.bfloat16)
    params[2].grad[3, 5] = float("nan")
    scao_amd.Muon(params).step()
    assert bool(params[2].isnan().all())
    assert not any(bool(p.isnan().any()) for i, p in enumerate(params) if i != 2)


def test_captured(hip_device):
    params, twin = _model(hip_device, torch.float32), _model(hip_device, torch.float32)
    a, b = scao_amd.Muon(params, lr=0.02), scao_amd.Muon(twin, lr=0.02)
    a.step()
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for k in range(3):
        for p, q in zip(params, twin):
            p.grad.copy_(torch.randn(p.shape, device=hip_device))
            q.grad.copy_(p.grad)
        graph.replay()
        b.step()
        assert all(torch.equal(p, q) for p, q in zip(params, twin))


def test_refusals(hip_device):
    w = torch.nn.Parameter(torch.zeros(4, 6, device=hip_device))
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(ns_steps=0),
                dict(eps=0.0), dict(adjust_lr_fn="x"), dict(ns_coefficients=(1.0, 2.0)),
                dict(ns_dtype=torch.float16)):
        with pytest.raises(ValueError):
            scao_amd.Muon([w], **bad)
    with pytest.raises(ValueError):
        scao_amd.Muon([torch.nn.Parameter(torch.zeros(4, device=hip_device))])
    opt = scao_amd.Muon([w])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(4, device=hip_device))]))
    assert len(opt.param_groups) == 1
    s = torch.nn.Parameter(torch.zeros(6, 4, device=hip_device).t())
    s.grad = torch.zeros_like(s)
    with pytest.raises(ValueError, match="contiguous"):
        scao_amd.Muon([s]).step()
    # two parameters of one memory
    buf = torch.zeros(8, 6, device=hip_device)
    ps = [torch.nn.Parameter(buf[:5]), torch.nn.Parameter(buf[4:])]
    for p in ps:
        p.grad = torch.ones_like(p)
    with pytest.raises(RuntimeError, match="share memory"):
        scao_amd.Muon(ps).step()

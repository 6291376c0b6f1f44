"""What the operators' shape functions refuse, over tensors without memory: no GPU
needed."""

from __future__ import annotations

import pytest
import torch

import scao_amd


def _heads(**kw):
    """arguments of qk_norm_rope's operator without memory, some of them others"""
    dim = kw.pop("dim", 64)
    args = dict(q=torch.empty(2, 4, 3, dim, device="meta"),
                k=torch.empty(2, 4, 1, dim, device="meta"), wq=None, wk=None,
                cos=torch.empty(4, 32, device="meta"), sin=torch.empty(4, 32, device="meta"),
                positions=None, eps=1e-6, interleaved=False)
    args.update(kw)
    return list(args.values())


def test_a_trace_refuses_the_heads_that_the_kernels_refuse():
    scao_amd._lib.torch_host()
    op, back = (torch.ops.scao_amd.qk_norm_rope, torch.ops.scao_amd.qk_norm_rope_backward)
    y = op(*_heads())
    assert [t.shape for t in back(*y, *_heads(), 3)] == [t.shape for t in y]
    none = torch.empty(2, 4, 0, 64, device="meta")
    for bad in (dict(dim=600), dict(dim=0), dict(q=none), dict(k=none), dict(eps=-1.0)):
        with pytest.raises(RuntimeError, match="qk_norm_rope"):
            op(*_heads(**bad))
        with pytest.raises(RuntimeError, match="qk_norm_rope"):
            back(*y, *_heads(**bad), 3)
    for gradients in ((y[1], y[1]), (y[0].double(), y[1]), (y[0], y[1][:1])):
        with pytest.raises(RuntimeError, match="gradients are not like"):
            back(*gradients, *_heads(), 3)
    with pytest.raises(RuntimeError, match="no weight"):
        back(*y, *_heads(), 4)


def test_a_trace_refuses_the_updates_that_the_kernels_refuse():
    scao_amd._lib.torch_host()
    op, co = torch.ops.scao_amd.orthogonalize, [1.5, -0.5, 0.0]
    m = torch.empty(8, 16, device="meta")
    assert op([m], co, 1e-7, torch.bfloat16)[0].dtype == torch.bfloat16
    assert op([torch.empty(0, 1 << 21, device="meta")], co, 1e-7, None)[0].shape == (0, 1 << 21)
    assert op([m], co, 1e-7, torch.float16, torch.float32)[0].dtype == torch.float16
    for args in (([m], co, 1e-7, None, torch.float16), ([m], co, 1e-7, torch.float64),
                 ([m.double()], co, 1e-7, None),
                 ([m[0]], co, 1e-7, None), ([m], co[:2], 1e-7, None), ([m], co * 65, 1e-7, None),
                 ([m], [], 1e-7, None), ([torch.empty(1 << 20, 4, device="meta")], co, 1e-7, None),
                 ([torch.empty(40000, 40000, device="meta")], co, 1e-7, None)):
        with pytest.raises(RuntimeError):
            op(*args)


def test_a_trace_refuses_the_steps_that_the_kernels_refuse():
    scao_amd._lib.torch_host()
    op = torch.ops.scao_amd.muon_step_
    p, m = torch.empty(8, 16, device="meta"), torch.empty(8, 16, device="meta")

    def step(params=(p,), grads=(p,), momenta=(m,), rates=(0.1,), decays=(1.0,), precisions=(0,)):
        op(list(params), list(grads), list(momenta), list(rates), list(decays), 0.9, True,
           [1.5, -0.5, 0.0], 1e-7, list(precisions))

    step()
    for bad in (dict(grads=()), dict(momenta=(m, m)), dict(rates=()), dict(decays=(1.0, 1.0)),
                dict(precisions=()), dict(momenta=(m.bfloat16(),)), dict(momenta=(m[:, :8],)),
                dict(grads=(p.t(),)), dict(grads=(p.double(),)),
                dict(params=(p.t(),), grads=(p.t(),), momenta=(m.t(),)),
                dict(params=(p[0],), grads=(p[0],), momenta=(m[0],))):
        with pytest.raises(RuntimeError):
            step(**bad)

"""Traces of the operators of include/scao_train.h over tensors without memory:
no GPU needed."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import scao_amd


def _ops(graph):
    return [str(n.target) for n in graph.graph.nodes if str(n.target).startswith("scao_amd.")]


def test_a_trace_holds_the_block():
    with FakeTensorMode():
        x, gate, up = (torch.empty(s, device="cuda", dtype=torch.bfloat16)
                       for s in ((3, 5, 16), (24, 16), (24, 16)))
        down = torch.empty(16, 24, device="cuda", dtype=torch.bfloat16)
        graph = make_fx(lambda *t: scao_amd.gated_ffn(*t))(x, gate, up, down)
        assert _ops(graph) == ["scao_amd.gated_ffn.default"]
        leaf = x.requires_grad_()
        y = scao_amd.gated_ffn(leaf, gate, up, down)
        assert y.shape == x.shape and y.device == x.device and y.requires_grad
        with pytest.raises(ValueError):
            scao_amd.gated_ffn(x, gate, up[:3], down)


def test_a_trace_holds_the_clipping():
    with FakeTensorMode():
        params = [torch.nn.Parameter(torch.empty(n, device="cuda")) for n in (7, 33)]

        def clip(*grads):
            for p, g in zip(params, grads):
                p.grad = g * 2
            norm = scao_amd.clip_grad_norm_(params, 0.5)
            return norm + scao_amd.global_grad_norm(params)

        graph = make_fx(clip)(*(torch.empty(n, device="cuda") for n in (7, 33)))
        assert _ops(graph) == ["scao_amd.grad_clip_.default", "scao_amd.grad_norm.default"]


def test_the_names_of_the_operators():
    scao_amd._lib.torch_host()
    for name in ("gated_ffn", "gated_ffn_save", "gated_ffn_backward", "grad_norm", "grad_clip_"):
        assert hasattr(torch.ops.scao_amd, name)

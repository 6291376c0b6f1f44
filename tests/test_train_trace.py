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


def test_the_names_of_the_operators():
    scao_amd._lib.torch_host()
    for name in ("gated_ffn", "gated_ffn_save", "gated_ffn_backward"):
        assert hasattr(torch.ops.scao_amd, name)

"""Traces of the orthogonalised updates and of the queries' and keys' norms over
tensors without memory: no GPU needed."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import scao_amd


def _ops(graph):
    return [str(n.target) for n in graph.graph.nodes if str(n.target).startswith("scao_amd.")]


def test_a_trace_holds_the_orthogonalisation():
    with FakeTensorMode():
        a, b = torch.empty(8, 16, device="cuda"), torch.empty(3, 5, 4, device="cuda")
        graph = make_fx(lambda *t: scao_amd.orthogonalize(list(t), dtype=torch.bfloat16))(a, b)
        assert _ops(graph) == ["scao_amd.orthogonalize.default"]
        out = scao_amd.orthogonalize([a, b])
        assert [t.shape for t in out] == [a.shape, b.shape] and out[0].dtype == torch.float32


def test_a_trace_holds_the_norms_and_rotation():
    with FakeTensorMode():
        q, k = (torch.empty(2, 6, h, 32, device="cuda", dtype=torch.bfloat16) for h in (4, 2))
        w = torch.empty(32, device="cuda")
        table = torch.empty(6, 16, device="cuda")
        graph = make_fx(lambda *t: scao_amd.qk_norm_rope(*t))(q, k, w, w, table, table)
        assert _ops(graph) == ["scao_amd.qk_norm_rope.default"]
        leaf = q.requires_grad_()
        y, yk = scao_amd.qk_norm_rope(leaf, k, w, w, table, table)
        assert y.shape == q.shape and yk.shape == k.shape and y.requires_grad
        with pytest.raises(ValueError):
            scao_amd.qk_norm_rope(q, k, w, w, table[:5], table[:5])


def test_a_trace_holds_the_step():
    with FakeTensorMode():
        params = [torch.nn.Parameter(torch.empty(s, device="cuda")) for s in ((8, 16), (2, 4, 4))]

        def step(*grads):
            for p, g in zip(params, grads):
                p.grad = g * 2
            scao_amd.Muon(params).step()
            return params[0] + 0

        graph = make_fx(step)(*(torch.empty(p.shape, device="cuda") for p in params))
        assert "scao_amd.muon_step_.default" in _ops(graph)


def test_the_names_of_the_operators():
    scao_amd._lib.torch_host()
    for name in ("orthogonalize", "muon_step_", "qk_norm_rope", "qk_norm_rope_backward"):
        assert hasattr(torch.ops.scao_amd, name)

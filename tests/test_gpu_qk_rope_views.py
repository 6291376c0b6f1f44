"""Queries and keys in views of any strides, overlapping ones among them: the same bits
as of contiguous copies, forward and backward."""

from __future__ import annotations

import pytest
import torch

import scao_amd
from tests.test_qk_rope_layouts import VIEWS, view

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("which", VIEWS)
def test_views(hip_device, which, dtype):
    g = torch.Generator(device=hip_device).manual_seed(3)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=hip_device).to(dtype)

    def pair():
        return view(normal(4, 1000), which), view(normal(4, 1000), which)[:, :, :1]

    inputs, gradients = pair(), pair()
    dim = inputs[0].shape[-1]
    weights = normal(dim), normal(dim)
    cos, sin = scao_amd.rotary_table(64, dim // 2 * 2, device=hip_device)

    def run(form):
        # (the leaves keep their strides: nothing copies them ahead of the operator)
        leaves = [form(t).detach().requires_grad_() for t in inputs]
        leaves += [w.clone().requires_grad_() for w in weights]
        alone = scao_amd.qk_norm_rope(*(t.detach() for t in leaves), cos, sin)
        y = scao_amd.qk_norm_rope(*leaves, cos, sin)
        return *alone, *y, *torch.autograd.grad(y, leaves, [form(t) for t in gradients])

    for a, b in zip(run(lambda t: t), run(lambda t: t.contiguous())):
        assert a.shape == b.shape and torch.equal(a, b)
        assert not bool(a.isnan().any())


@pytest.mark.parametrize("which", VIEWS)
def test_a_trace_says_how_outputs_lie(hip_device, which):
    scao_amd._lib.torch_host()
    x = torch.randn(4, 1000, device=hip_device)
    strides = []
    for t in (x, x.to("meta")):
        q = view(t, which)
        table = torch.ones(64, q.shape[-1] // 2, device=t.device)
        rest = q, q, None, None, table, table, None, 1e-6, False
        y = torch.ops.scao_amd.qk_norm_rope(*rest)
        dx = torch.ops.scao_amd.qk_norm_rope_backward(q, q, *rest, 3)
        strides.append([o.stride() for o in (*y, *dx)])
    assert strides[0] == strides[1]


def test_vmapped(hip_device):
    """torch maps the operator over a dimension by calling it for every entry."""
    q = torch.randn(3, 2, 5, 4, 32, device=hip_device)
    w = torch.randn(3, 32, device=hip_device)
    cos, sin = scao_amd.rotary_table(5, 32, device=hip_device)
    got = torch.func.vmap(lambda a, b: scao_amd.qk_norm_rope(a, a[:, :, :1], b, b, cos, sin))(q, w)
    for i in range(3):
        one = scao_amd.qk_norm_rope(q[i], q[i, :, :, :1], w[i], w[i], cos, sin)
        assert all(torch.equal(a[i], b) for a, b in zip(got, one))
    # what torch cannot map is refused
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda a: scao_amd.orthogonalize(a))(q[:, 0, 0])
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: scao_amd.qk_norm_rope(a, a, None, None, cos, sin)[0].sum())(q[0])

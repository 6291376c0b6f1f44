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

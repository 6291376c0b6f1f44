"""How the outputs of the queries' and keys' norms lie in memory, from tensors without
memory: no GPU needed.  The kernels write columns of unit stride."""

from __future__ import annotations

import pytest
import torch

import scao_amd

VIEWS = {
    "windows as tokens": lambda x: x[:1, :67].unfold(1, 64, 1).unsqueeze(2),
    "windows as sequences": lambda x: x[0, :67].unfold(0, 64, 1).unsqueeze(1).unsqueeze(2),
    "windows as heads": lambda x: x[:2, :70].unfold(1, 64, 1).unsqueeze(1),
    "windows of windows": lambda x: x[:2, :54].unfold(1, 8, 1).unfold(1, 2, 3).permute(0, 1, 3, 2),
    "one column apart": lambda x: x.as_strided((2, 2, 3, 8), (27, 1, 9, 1)),
    "sequences and tokens alike": lambda x: x.as_strided((3, 4, 2, 16), (1, 1, 1, 1)),
    "expanded": lambda x: x[0, :64].expand(2, 3, 4, 64),
    "slices of wider rows": lambda x: x[:2, :960].unflatten(1, (3, 5, 64))[:, :, 1:3],
    "heads before tokens": lambda x: x[:2, :960].unflatten(1, (3, 5, 64)).transpose(1, 2),
    "columns before heads": lambda x: x[:2, :960].unflatten(1, (3, 64, 5)).transpose(2, 3),
    "every other column": lambda x: x[:2, :960].unflatten(1, (3, 5, 64)).transpose(1, 2)[..., ::2],
    "one column": lambda x: x[:2, :12].unflatten(1, (3, 4, 1)).transpose(1, 2),
}


def view(x, which):
    """one of VIEWS of x (4 x 1000), as (batch, tokens, heads, columns)"""
    return VIEWS[which](x)


@pytest.mark.parametrize("which", VIEWS)
def test_outputs_have_unit_columns(which):
    scao_amd._lib.torch_host()
    q = view(torch.empty(4, 1000, device="meta"), which)
    half = q.shape[-1] // 2
    table = torch.empty(64, half, device="meta")
    y = torch.ops.scao_amd.qk_norm_rope(q, q, None, None, table, table, None, 1e-6, False)
    dx = torch.ops.scao_amd.qk_norm_rope_backward(*y, q, q, None, None, table, table, None, 1e-6,
                                                  False, 3)
    for t in (*y, *dx):
        assert t.shape == q.shape
        assert t.stride(-1) == 1 or t.shape[-1] == 1
        # no two elements of one place
        assert torch._prims_common.is_non_overlapping_and_dense(t)


@pytest.mark.parametrize("which", ["columns before heads", "every other column"])
def test_copied_inputs_have_contiguous_outputs(which):
    """Columns of another stride are copied ahead of the kernels, which is what a trace has
    to say of their outputs."""
    scao_amd._lib.torch_host()
    q = view(torch.empty(4, 1000, device="meta"), which)
    assert q.stride(-1) != 1
    table = torch.empty(8, 16, device="meta")
    y = torch.ops.scao_amd.qk_norm_rope(q, q, None, None, table, table, None, 1e-6, False)
    dx = torch.ops.scao_amd.qk_norm_rope_backward(*y, q, q, None, None, table, table, None, 1e-6,
                                                  False, 3)
    for t in (*y, *dx):
        assert t.shape == q.shape and t.is_contiguous()

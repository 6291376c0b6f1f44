"""GatedFFN without a GPU: its weights."""

from __future__ import annotations

import pytest

import scao_amd


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("d_model,d_ff", [(8, 0), (0, 8), (0, 0), (8, 24)])
def test_sizes_of_the_weights(d_model, d_ff, packed):
    """Sizes of zero too, which the block takes."""
    m = scao_amd.GatedFFN(d_model, d_ff, packed=packed)
    shapes = {k: tuple(p.shape) for k, p in m.named_parameters()}
    assert shapes.pop("down") == (d_model, d_ff)
    assert shapes == ({"gate_up": (2 * d_ff, d_model)} if packed else
                      {"gate": (d_ff, d_model), "up": (d_ff, d_model)})
    for p in m.parameters():
        assert not p.numel() or p.abs().max().item() <= p.shape[1] ** -0.5

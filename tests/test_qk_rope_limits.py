"""How many heads one call of the queries' and keys' norms takes: refused on the host, no
GPU needed."""

from __future__ import annotations

import pytest

from scao_amd import _lib as L
from tests.test_ortho_rope_capi import _rope, _tensors


@pytest.mark.parametrize("dim,dtype,lanes", [(512, 0, 64), (129, 1, 64), (128, 1, 8)])
def test_more_lanes_than_a_launch_has(dim, dtype, lanes):
    """2^32 threads: lanes a group, a group for queries and one for keys"""
    tokens = (1 << 32) // (2 * lanes)
    lib = L.lib()
    for seq, what in ((tokens, b"lanes"), (tokens * 2, b"lanes")):
        t, y = _rope(dim=dim, dtype=dtype, heads=(1, 1), batch=1, seq=seq), _tensors()
        assert lib.scao_qk_rope_forward(t.ctypes.data, y.ctypes.data, None) == 1
        assert what in lib.scao_last_error()

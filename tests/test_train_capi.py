"""The C ABI of include/scao_train.h without a GPU: every declared symbol is
exported and bound, and bad arguments are refused on the host, with the entry
point's name in the message, before anything is launched."""

from __future__ import annotations

import ctypes
import os
import re

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "scao_train.h")

P = 16   # a non-null, aligned dummy address: nothing is launched


def _declared():
    txt = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return sorted(set(re.findall(r"\b(scao_[a-z0-9_]+)\s*\(", txt)))


def test_library_exports_every_declared_symbol():
    from scao_amd import _lib as L
    lib = L.lib()
    assert sorted(L.TRAIN_SIGNATURES) == _declared()
    for n in _declared():
        assert hasattr(lib, n)


def _table(*rows):
    from scao_amd import _lib as L
    t = np.zeros(len(rows), dtype=L.TENSOR_DESC)
    for i, (data, numel, dtype) in enumerate(rows):
        t[i] = (data, numel, dtype, 0)
    return t


GOOD = [(4096, 10, 0)]
BAD_CLIP = [
    # table rows, norm type, scale, max_norm, norm, workspace
    (None, 2, 1.0, 1.0, P, P),
    (GOOD, 3, 1.0, 1.0, P, P),
    (GOOD, -1, 1.0, 1.0, P, P),
    (GOOD, 2, 0.0, 1.0, P, P),
    (GOOD, 2, float("nan"), 1.0, P, P),
    (GOOD, 2, float("inf"), 1.0, P, P),
    (GOOD, 2, 1.0, 1.0, None, P),
    (GOOD, 2, 1.0, 1.0, P, None),
    ([(0, 10, 0)], 2, 1.0, 1.0, P, P),
    ([(4098, 10, 0)], 2, 1.0, 1.0, P, P),
    ([(4097, 10, 1)], 2, 1.0, 1.0, P, P),
    ([(4096, -1, 0)], 2, 1.0, 1.0, P, P),
    ([(4096, 10, 3)], 2, 1.0, 1.0, P, P),
    ([(1 << 57, 10, 0)], 2, 1.0, 1.0, P, P),   # no address
]


@pytest.mark.parametrize("rows,kind,scale,max_norm,norm,work", BAD_CLIP)
def test_norm_and_clip_refuse_bad_arguments(rows, kind, scale, max_norm, norm, work):
    from scao_amd import _lib as L
    lib = L.lib()
    t = _table(*rows) if rows else None
    at = t.ctypes.data if rows else None
    assert lib.scao_grad_norm(at, 1, kind, scale, norm, work, None) == 1
    assert lib.scao_last_error().startswith(b"scao_grad_norm:")
    assert lib.scao_grad_clip(at, 1, kind, scale, max_norm, norm, work, None) == 1
    assert lib.scao_last_error().startswith(b"scao_grad_clip:")


def test_clip_refuses_bad_bounds_and_shared_memory():
    from scao_amd import _lib as L
    lib = L.lib()
    t = _table(*GOOD)
    for max_norm in (-1.0, float("nan")):
        assert lib.scao_grad_clip(t.ctypes.data, 1, 2, 1.0, max_norm, P, P, None) == 1
    for rows in ([(4096, 10, 0), (4096, 10, 0)], [(4132, 4, 0), (4096, 10, 0)],
                 [(4096, 10, 1), (8192, 1, 0), (4114, 5, 1)]):
        t = _table(*rows)
        assert lib.scao_grad_clip(t.ctypes.data, len(rows), 2, 1.0, 1.0, P, P, None) == 1
        assert b"share memory" in lib.scao_last_error()


def test_workspace_holds_every_launch():
    from scao_amd import _lib as L
    lib = L.lib()
    t = _table(*GOOD * 400)
    assert lib.scao_grad_norm_workspace(t.ctypes.data, 0) == 0
    assert lib.scao_grad_norm_workspace(t.ctypes.data, 1) == 2048 * 8
    assert lib.scao_grad_norm_workspace(t.ctypes.data, 400) == 2 * 2048 * 8


def _ffn(**kw):
    from scao_amd import _lib as L
    base = dict(x=4096, w_gate=4096, w_up=4096, w_down=4096, ldx=16, ld_gate=16, ld_up=16,
                ld_down=24, tokens=3, d=16, f=24, dtype=1, act=0)
    base.update(kw)
    t = np.zeros(1, dtype=L.FFN_DESC)
    for k, v in base.items():
        t[k] = v
    return t


BAD_FFN = [dict(x=0), dict(w_gate=0), dict(w_up=4097), dict(w_down=0), dict(ldx=15),
           dict(ld_gate=15), dict(ld_up=8), dict(ld_down=23), dict(ldx=1 << 21), dict(tokens=0),
           dict(tokens=-1), dict(tokens=1 << 31), dict(d=0), dict(d=1 << 21), dict(f=0),
           dict(f=1 << 20), dict(dtype=3), dict(dtype=-1), dict(act=5), dict(act=-1),
           dict(x=4098, dtype=0)]


@pytest.mark.parametrize("kw", BAD_FFN)
def test_ffn_refuses_bad_descriptors(kw):
    from scao_amd import _lib as L
    lib = L.lib()
    t = _ffn(**kw)
    at = t.ctypes.data
    assert lib.scao_ffn_forward(at, P, None, P, None) == 1
    assert lib.scao_last_error().startswith(b"scao_ffn_forward:")
    assert lib.scao_ffn_backward(at, P, 16, P, P, P, P, P, P, None) == 1
    assert lib.scao_last_error().startswith(b"scao_ffn_backward:")
    assert lib.scao_ffn_forward_workspace(at, 0) == 0
    assert lib.scao_ffn_backward_workspace(at, P, 16, 15) == 0


def test_ffn_refuses_bad_buffers():
    from scao_amd import _lib as L
    lib = L.lib()
    t = _ffn()
    at = t.ctypes.data
    assert lib.scao_ffn_forward(None, P, None, P, None) == 1
    assert lib.scao_ffn_backward(None, P, 16, P, P, P, P, P, P, None) == 1
    for y, saved, work in ((None, None, P), (17, None, P), (P, 8, P), (P, None, 8), (P, None, None)):
        assert lib.scao_ffn_forward(at, y, saved, work, None) == 1
    for args in ((None, 16, P, P, P, P, P, P), (P, 15, P, P, P, P, P, P),
                 (P, 16, None, P, P, P, P, P), (P, 16, P, P, P, P, P, None),
                 (P, 16, P, 17, P, P, P, P), (P, 16, P, P, P, P, 17, P)):
        assert lib.scao_ffn_backward(at, *args, None) == 1


def test_ffn_sizes_of_buffers():
    """h, a and b: what the header's formulas need and no packing for operands
    that can be loaded as they are."""
    from scao_amd import _lib as L
    lib = L.lib()
    t = _ffn(tokens=32, d=64, f=48, ldx=64, ld_gate=64, ld_up=64, ld_down=48)
    frags = 2 * 3
    assert lib.scao_ffn_saved_bytes(t.ctypes.data) == 32 * 48 * 2 + frags * 64 * 24
    assert lib.scao_ffn_forward_workspace(t.ctypes.data, 1) == 0
    assert lib.scao_ffn_forward_workspace(t.ctypes.data, 0) == 32 * 48 * 2
    t = _ffn(tokens=32, d=64, f=48, ldx=64, ld_gate=64, ld_up=64, ld_down=48, dtype=0)
    assert lib.scao_ffn_saved_bytes(t.ctypes.data) == 3 * 32 * 48 * 2 + frags * 64 * 32
    assert lib.scao_ffn_forward_workspace(t.ctypes.data, 1) >= 3 * 2 * (32 * 64 + 3 * 64 * 48)

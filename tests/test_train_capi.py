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
    assert lib.scao_grad_norm_workspace(t.ctypes.data, 400) == 3 * 2048 * 8

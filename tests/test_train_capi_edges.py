"""What the C ABI of include/scao_train.h accepts at its ends, without a GPU:
nothing is launched."""

from __future__ import annotations

import numpy as np


def _ffn(**kw):
    from scao_amd import _lib as L
    t = np.zeros(1, dtype=L.FFN_DESC)
    base = dict(x=4096, w_gate=4096, w_up=4096, w_down=4096, ldx=16, ld_gate=16, ld_up=16,
                ld_down=24, tokens=3, d=16, f=24, dtype=1, act=0)
    for k, v in {**base, **kw}.items():
        t[k] = v
    return t


def test_the_stride_of_a_single_row_is_not_looked_at():
    from scao_amd import _lib as L
    lib = L.lib()
    for stride in (0, 1 << 21, 1 << 40):
        for kw in (dict(tokens=1, ldx=stride), dict(f=1, ld_gate=stride), dict(f=1, ld_up=stride),
                   dict(d=1, ld_down=stride)):
            t = _ffn(**kw)
            assert lib.scao_ffn_forward_workspace(t.ctypes.data, 0) > 0, kw
            assert lib.scao_ffn_backward_workspace(t.ctypes.data, 4096, 16, 15) > 0, kw
            many = _ffn(**{k: v for k, v in kw.items() if k.startswith("ld")})
            assert lib.scao_ffn_forward_workspace(many.ctypes.data, 0) == 0
            assert b"row stride" in lib.scao_last_error()


def test_buffers_off_their_alignment_are_refused():
    from scao_amd import _lib as L
    lib = L.lib()
    t = np.zeros(1, dtype=L.TENSOR_DESC)
    t[0] = (4096, 10, 0, 0)
    for norm, work in ((4, 4), (4, 12), (2, 8), (5, 16)):
        assert lib.scao_grad_norm(t.ctypes.data, 1, 2, 1.0, norm, work, None) == 1
        assert b"not aligned" in lib.scao_last_error()
        assert lib.scao_grad_clip(t.ctypes.data, 1, 2, 1.0, 1.0, norm, work, None) == 1
        assert b"not aligned" in lib.scao_last_error()

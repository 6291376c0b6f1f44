"""The C ABI of the orthogonalised updates and of the queries' and keys' norms
without a GPU: bad arguments are refused on the host, with the entry point's name in
the message, before anything is launched; and what Python refuses there."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import scao_amd
from scao_amd import _lib as L

P = 4096   # a non-null, aligned dummy address: nothing is launched
CO = np.array([1.5, -0.5, 0.0] * 2)


def _ortho(sizes=(200,), **kw):
    t = np.zeros(len(sizes), dtype=L.ORTHO_DESC)
    for i, m in enumerate(sizes):
        base = dict(src=P + (i << 24), dst=(1 << 40) + (i << 24), rows=m, cols=300, ld_src=300,
                    ld_dst=300, src_dtype=1, dst_dtype=1)
        base.update(kw)
        for k, v in base.items():
            t[i][k] = v
    return t


def _muon(**kw):
    t = np.zeros(1, dtype=L.MUON_DESC)
    base = dict(p=P, g=1 << 40, m=1 << 41, rows=200, cols=300, dtype=1, grad_dtype=1, rate=0.1,
                decay=1.0)
    base.update(kw)
    for k, v in base.items():
        t[0][k] = v
    return t


def _call(t, coefficients=CO, steps=2, eps=1e-7, work=P, momentum=None, n=None):
    at, co = t.ctypes.data, coefficients.ctypes.data if coefficients is not None else None
    n = len(t) if n is None else n
    if momentum is None:
        return L.lib().scao_orthogonalize(at, n, co, steps, eps, work, None)
    return L.lib().scao_muon_step(at, n, momentum, 1, co, steps, eps, work, None)


BAD_SCHEME = [dict(steps=0), dict(steps=65), dict(coefficients=None), dict(eps=0.0),
              dict(eps=1e-310),
              dict(eps=float("nan")), dict(coefficients=np.array([np.inf] * 6)), dict(n=-1),
              dict(work=P + 8), dict(work=None),
              # 40^2 > 1024
              dict(coefficients=np.array([40.0, 0.0, 0.0] * 2))]


@pytest.mark.parametrize("bad", BAD_SCHEME)
def test_schemes_are_refused(bad):
    assert _call(_ortho(), **bad) == 1
    assert L.lib().scao_last_error().startswith(b"scao_orthogonalize:")
    assert _call(_muon(), momentum=0.9, **bad) == 1
    assert L.lib().scao_last_error().startswith(b"scao_muon_step:")


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(cols=1 << 20), dict(rows=40000, cols=40000),
                                 dict(src_dtype=3), dict(dst_dtype=-1), dict(src=0), dict(dst=0),
                                 dict(src=P + 1), dict(ld_src=299), dict(ld_dst=1 << 31),
                                 dict(precision=2), dict(dst=P)])
def test_matrices_are_refused(bad):
    t = _ortho(**bad)
    if "cols" in bad:
        t["ld_src"] = t["ld_dst"] = t["cols"]
    assert _call(t) == 1
    assert L.lib().scao_last_error().startswith(b"scao_orthogonalize:")


@pytest.mark.parametrize("bad", [dict(p=0), dict(g=0), dict(m=0), dict(m=(1 << 41) + 2),
                                 dict(p=(1 << 41) + 64), dict(rate=float("nan")),
                                 dict(decay=float("inf")), dict(grad_dtype=7), dict(precision=-1)])
def test_parameters_are_refused(bad):
    assert _call(_muon(**bad), momentum=0.9) == 1
    assert L.lib().scao_last_error().startswith(b"scao_muon_step:")


def test_momentum_is_refused():
    for mu in (-0.1, 1.0, float("nan")):
        assert _call(_muon(), momentum=mu) == 1


def test_shared_memory_is_refused():
    t = _ortho(sizes=(200, 200))
    t[1]["dst"] = int(t[0]["dst"]) + 200 * 300 * 2 - 2
    assert _call(t) == 1 and b"share memory" in L.lib().scao_last_error()
    t[1]["dst"] = int(t[0]["src"]) + 64
    assert _call(t) == 1 and b"share memory" in L.lib().scao_last_error()


def test_workspaces():
    lib = L.lib()
    assert lib.scao_orthogonalize_workspace(None, 0, 5) == 0
    # matrices that one workgroup holds need none
    small = _ortho(sizes=(50, 60), cols=64, ld_src=64, ld_dst=64)
    assert lib.scao_orthogonalize_workspace(small.ctypes.data, 2, 5) == 0
    one = _ortho(sizes=(600,))
    need = lib.scao_orthogonalize_workspace(one.ctypes.data, 1, 5)
    # X twice (but for one step), A and B, 16 bits each
    least = 2 * 600 * 304 * 2 + 2 * 300 * 304 * 2
    assert need >= least
    assert lib.scao_orthogonalize_workspace(one.ctypes.data, 1, 1) <= need - 600 * 304 * 2
    one["precision"] = 1
    assert lib.scao_orthogonalize_workspace(one.ctypes.data, 1, 5) >= 2 * least
    # a pass does not grow with the model: 64 matrices, as many as 400
    many, more = _ortho(sizes=(600,) * 64), _ortho(sizes=(600,) * 400)
    assert lib.scao_orthogonalize_workspace(more.ctypes.data, 400, 5) == \
        lib.scao_orthogonalize_workspace(many.ctypes.data, 64, 5)


def _rope(**kw):
    t = np.zeros(1, dtype=L.ROPE_DESC)
    base = dict(cos=P, sin=P, batch=2, seq=3, table_rows=8, ld_table=16, heads=(4, 2), dim=64,
                rotary=32, dtype=1, eps=1e-6)
    base.update(kw)
    for k, v in base.items():
        t[0][k] = v
    t[0]["x"]["p"] = P
    return t


def _tensors(p=P):
    t = np.zeros(2, dtype=L.ROPE_TENSOR)
    t["p"] = p
    return t


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(dim=0), dict(dim=513), dict(rotary=66),
                                 dict(rotary=31), dict(heads=(0, 2)), dict(heads=(4, 1 << 16)),
                                 dict(batch=-1), dict(seq=1 << 31), dict(batch=1 << 20, seq=1 << 12),
                                 dict(eps=-1.0), dict(eps=float("nan")), dict(cos=0),
                                 dict(sin=P + 2), dict(ld_table=15), dict(w=(P + 1, 0)),
                                 dict(w=(0, P), w_dtype=(0, 5)),
                                 dict(positions=P + 4, wide_positions=1)])
def test_heads_are_refused(bad):
    t, y = _rope(**bad), _tensors()
    lib = L.lib()
    assert lib.scao_qk_rope_forward(t.ctypes.data, y.ctypes.data, None) == 1
    assert lib.scao_last_error().startswith(b"scao_qk_rope_forward:")
    assert lib.scao_qk_rope_backward(t.ctypes.data, y.ctypes.data, y.ctypes.data, None, None, P,
                                     None) == 1
    assert lib.scao_last_error().startswith(b"scao_qk_rope_backward:")


def test_tensors_of_heads_are_refused():
    lib, t, y = L.lib(), _rope(), _tensors()
    for bad in (0, P + 1):
        z = _tensors(bad)
        assert lib.scao_qk_rope_forward(t.ctypes.data, z.ctypes.data, None) == 1
        assert lib.scao_qk_rope_backward(t.ctypes.data, z.ctypes.data, y.ctypes.data, None, None,
                                         P, None) == 1
    # a weight's gradient without the weight, without a workspace, off its alignment
    at = y.ctypes.data
    assert lib.scao_qk_rope_backward(t.ctypes.data, at, at, P, None, P, None) == 1
    t = _rope(w=(P, P), w_dtype=(1, 1))
    assert lib.scao_qk_rope_backward(t.ctypes.data, at, at, P, P, None, None) == 1
    assert lib.scao_qk_rope_backward(t.ctypes.data, at, at, P + 1, P, P, None) == 1
    assert lib.scao_qk_rope_forward(None, at, None) == 1
    assert lib.scao_qk_rope_forward(t.ctypes.data, None, None) == 1


def test_the_backward_pass_has_room_for_every_workgroup():
    lib = L.lib()
    for batch, seq in ((1, 1), (2, 3), (64, 4096)):
        t = _rope(batch=batch, seq=seq)
        need = lib.scao_qk_rope_backward_workspace(t.ctypes.data)
        assert need % (2 * 64 * 4) == 0 and 1 <= need // (2 * 64 * 4) <= 768
    assert lib.scao_qk_rope_backward_workspace(_rope(seq=0).ctypes.data) == 0


def test_python_refuses_tensors_off_the_gpu():
    m = torch.zeros(4, 4)
    with pytest.raises(RuntimeError):
        scao_amd.orthogonalize(m)
    cos, sin = scao_amd.rotary_table(4, 4)
    q = torch.zeros(1, 2, 3, 4)
    with pytest.raises(RuntimeError):
        scao_amd.qk_norm_rope(q, q, None, None, cos, sin)
    p = torch.nn.Parameter(m)
    p.grad = m
    with pytest.raises(RuntimeError):
        scao_amd.Muon([p]).step()


@pytest.mark.parametrize("kw", [dict(steps=0), dict(steps=2.5), dict(coefficients=(1.0, 2.0)),
                                dict(coefficients=[(1.0, 2.0, 3.0)] * 4), dict(eps=-1.0),
                                dict(eps=1e-310),
                                dict(coefficients=(1.0, float("nan"), 0.0))])
def test_python_refuses_schemes(kw):
    with pytest.raises(ValueError):
        scao_amd.orthogonalize(torch.zeros(4, 4), **kw)


def test_rotary_table():
    cos, sin = scao_amd.rotary_table(200001, 8, 500000.0)
    i = torch.arange(4, dtype=torch.float64)
    want = 200000.0 * 500000.0 ** (-2 * i / 8)
    assert cos.shape == (200001, 4) and cos.dtype == torch.float32
    assert torch.equal(cos[-1], torch.cos(want).float())
    assert torch.equal(sin[-1], torch.sin(want).float())
    assert scao_amd.rotary_table(3, 0)[0].shape == (3, 0)
    for bad in ((-1, 4), (4, 3), (4, -2)):
        with pytest.raises(ValueError):
            scao_amd.rotary_table(*bad)
    with pytest.raises(ValueError):
        scao_amd.rotary_table(4, 4, base=0.0)


def test_muon_momentum_keeps_its_bits_through_a_checkpoint():
    def make(seed):
        torch.manual_seed(seed)
        return [torch.nn.Parameter(torch.randn(3, 5).bfloat16()) for _ in range(2)]

    a, b = scao_amd.Muon(make(0)), scao_amd.Muon(make(1), lr=0.7)
    for p in a.param_groups[0]["params"]:
        a.state[p]["momentum_buffer"] = torch.randn(3, 5)
    b.load_state_dict(a.state_dict())
    for p, q in zip(a.param_groups[0]["params"], b.param_groups[0]["params"]):
        x, y = a.state[p]["momentum_buffer"], b.state[q]["momentum_buffer"]
        assert torch.equal(x, y) and y.dtype == torch.float32 and x.data_ptr() != y.data_ptr()
    assert b.param_groups[0]["lr"] == a.param_groups[0]["lr"]

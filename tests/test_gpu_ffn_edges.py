"""The feed-forward block at the ends of what it takes: infinite
pre-activations, rows of any stride, sizes of one, tracing, forward mode.

Where a call is compared with the same call on contiguous copies the bits have
to be equal; everything else has an exact result (zero or NaN)."""

from __future__ import annotations

import math

import pytest
import torch

import scao_amd

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _normal(dev, seed, *shape, dtype=torch.bfloat16, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * std).to(dtype)


def _inputs(dev, tokens, d, f, dtype=torch.bfloat16):
    return [_normal(dev, 0, tokens, d, dtype=dtype),
            _normal(dev, 1, f, d, dtype=dtype, std=d ** -0.5),
            _normal(dev, 2, f, d, dtype=dtype, std=d ** -0.5),
            _normal(dev, 3, d, f, dtype=dtype, std=f ** -0.5),
            _normal(dev, 4, tokens, d, dtype=dtype)]


def _run(x, gate, up, down, dy, name="silu"):
    leaves = [t.detach().requires_grad_() for t in (x, gate, up, down)]
    y = scao_amd.gated_ffn(*leaves, activation=name)
    grads = torch.autograd.grad(y, leaves, dy)
    return dict(y=y.detach(), **dict(zip(("dx", "dgate", "dup", "ddown"), grads)))


def _same(got, want):
    for k in want:
        assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,d,f", [(5, 8, 16), (33, 41, 53), (300, 72, 130)])
def test_relu_of_minus_infinity_is_zero(hip_device, dtype, tokens, d, f):
    """Every pre-activation is minus infinity: from a sum that overflows (fp32,
    bf16; powers of two, whose split parts are zero) or from a weight (16-bit)."""
    x, gate, up, down, dy = _inputs(hip_device, tokens, d, f, dtype)
    up[:, 0] = 0
    for large in ([2.0 ** 80] if dtype != torch.float16 else []) + \
                 ([math.inf] if dtype != torch.float32 else []):
        x[:, 0] = 1.0 if math.isinf(large) else large
        gate[:, 0] = -large
        got = _run(x, gate, up, down, dy, "relu")
        got["forward"] = scao_amd.gated_ffn(x, gate, up, down, "relu")
        if math.isinf(large):
            del got["dx"]   # 0 * infinity
        for k, v in got.items():
            assert bool(v.eq(0).all()), (k, large)
    x[tokens // 2, 1] = math.nan
    y = scao_amd.gated_ffn(x, gate, up, down, "relu")
    assert bool(y[tokens // 2].isnan().all()) and int(y.isnan().sum()) == d


def _wide(t, stride):
    """t's values in rows that begin `stride` elements apart"""
    out = torch.zeros(t.shape[0] * stride, dtype=t.dtype, device=t.device).view(-1, stride)
    out[:, :t.shape[1]] = t
    return out[:, :t.shape[1]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,d,f", [(1, 64, 24), (3, 64, 24), (70, 33, 9)])
def test_rows_of_any_stride(hip_device, dtype, tokens, d, f):
    """Rows 2^21 elements and more apart, in every matrix and in dy, and the
    last token of a long prompt."""
    ins = _inputs(hip_device, tokens, d, f, dtype)
    want, forward = _run(*ins), scao_amd.gated_ffn(*ins[:4])
    for i in range(5):
        moved = list(ins)
        moved[i] = _wide(ins[i], (1 << 21) + 8 * i)
        _same(_run(*moved), want)
        if i < 4:
            assert torch.equal(scao_amd.gated_ffn(*moved[:4]), forward)
    hidden = torch.zeros(tokens, (1 << 21) // 64, 64, dtype=dtype, device=hip_device)[:, :, :d]
    hidden[:, -1] = ins[0]
    assert torch.equal(scao_amd.gated_ffn(hidden[:, -1], *ins[1:4]), forward)


def test_outputs_taken_from_a_long_sequence(hip_device):
    """The gradient of the output arrives as rows of a much larger one."""
    ins = _inputs(hip_device, 3, 64, 24)
    want = _run(*ins)
    leaves = [t.detach().requires_grad_() for t in ins[:4]]
    y = scao_amd.gated_ffn(*leaves)
    long = torch.zeros(3, (1 << 21) // 64, 64, dtype=y.dtype, device=hip_device)
    grads = torch.autograd.grad(torch.cat([y[:, None], long], 1), leaves,
                                torch.cat([ins[4][:, None], long], 1))
    _same(dict(zip(("dx", "dgate", "dup", "ddown"), grads)),
          {k: v for k, v in want.items() if k != "y"})


def _column(t):
    """a tensor of one column whose column stride is not one"""
    return t.t().contiguous().t() if t.shape[1] == 1 else t


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,d,f", [(5, 1, 7), (5, 7, 1), (70, 1, 9), (1, 1, 1)])
def test_single_columns_of_any_stride(hip_device, dtype, tokens, d, f):
    """Torch ignores the stride of a dimension of one, and calls such a tensor
    contiguous whatever it is."""
    ins = _inputs(hip_device, tokens, d, f, dtype)
    want, forward = _run(*ins), scao_amd.gated_ffn(*ins[:4])
    odd = [_column(t).as_strided(t.shape, (1, 5)) if t.shape[1] == 1 else t for t in ins]
    assert any(t.stride(1) == 5 for t in odd)
    assert all(torch.equal(a, b) for a, b in zip(odd, ins))
    _same(_run(*odd), want)
    assert torch.equal(scao_amd.gated_ffn(*odd[:4]), forward)


def test_traces_hold_the_block(hip_device):
    """A trace computes the block of the inputs that it is called with."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, gate, up, down, dy = _inputs(hip_device, 20, 24, 40)
    new = _normal(hip_device, 7, 20, 24)

    def forward(x):
        return scao_amd.gated_ffn(x, gate, up, down)

    def training(x, dy):
        leaves = [t.detach().requires_grad_() for t in (x, gate, up, down)]
        return torch.autograd.grad(scao_amd.gated_ffn(*leaves), leaves, dy)

    for traced in (torch.jit.trace(forward, (x,)), make_fx(forward)(x)):
        assert torch.equal(traced(new), forward(new))
    traced = make_fx(training)(x, dy)
    for got, want in zip(traced(new, 2 * dy), training(new, 2 * dy)):
        assert torch.equal(got, want)


def test_dispatch_modes_see_the_block(hip_device):
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    ins = _inputs(hip_device, 20, 24, 40)
    want = _run(*ins)
    with Log():
        scao_amd.gated_ffn(*ins[:4])
        got = _run(*ins)
    _same(got, want)
    assert {s.split(".")[1] for s in seen if s.startswith("scao_amd.")} == {
        "gated_ffn", "gated_ffn_save", "gated_ffn_backward"}


def test_operators_check_their_arguments(hip_device):
    """Called by their names, past the Python function's own checks."""
    x, gate, up, down, dy = _inputs(hip_device, 20, 24, 40)
    scao_amd.gated_ffn(x, gate, up, down)
    op = torch.ops.scao_amd.gated_ffn
    assert torch.equal(op(x, gate, up, down, 0), scao_amd.gated_ffn(x, gate, up, down))
    for bad in ((x, gate, up[:-1], down, 0), (x[:, :-1], gate, up, down, 0),
                (x, gate, up, down.t(), 0), (x[0], gate, up, down, 0),
                (x.float(), gate, up, down, 0), (x, gate, up, down, 5),
                (x, gate, up, down.cpu(), 0), (x.double(),) * 4 + (0,)):
        with pytest.raises(RuntimeError):
            op(*bad)
    y, saved = torch.ops.scao_amd.gated_ffn_save(x, gate, up, down, 0)
    back = torch.ops.scao_amd.gated_ffn_backward
    assert len(back(dy, saved, x, gate, up, down, 0, 15)) == 4
    for bad in ((dy[:-1], saved), (dy, saved[:-1]), (dy, saved.cpu()), (dy.float(), saved)):
        with pytest.raises(RuntimeError):
            back(*bad, x, gate, up, down, 0, 15)


def test_negated_views(hip_device):
    """Tensors that hold their values negated, as the imaginary part of a
    conjugate does."""
    ins = _inputs(hip_device, 20, 24, 40)
    want, forward = _run(*ins), scao_amd.gated_ffn(*ins[:4])
    for i in range(5):
        moved = list(ins)
        moved[i] = torch._neg_view(-ins[i])
        assert moved[i].is_neg()
        _same(_run(*moved), want)
        if i < 4:
            assert torch.equal(scao_amd.gated_ffn(*moved[:4]), forward)


def test_traces_without_memory(hip_device):
    """A trace of shapes alone, and its run on real tensors."""
    from torch.fx.experimental.proxy_tensor import make_fx
    ins = _inputs(hip_device, 20, 24, 40)

    def training(x, gate, up, down, dy):
        leaves = [t.detach().requires_grad_() for t in (x, gate, up, down)]
        y = scao_amd.gated_ffn(*leaves)
        return y.detach(), *torch.autograd.grad(y, leaves, dy)

    want = _run(*ins)
    for mode in ("fake", "symbolic"):
        traced = make_fx(training, tracing_mode=mode)(*ins)
        for got, k in zip(traced(*ins), want):
            assert torch.equal(got, want[k]), mode


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(hip_device, which, grad):
    import torch.autograd.forward_ad as fwd
    ins = [t.requires_grad_(grad) for t in _inputs(hip_device, 20, 24, 40)[:4]]
    with fwd.dual_level():
        ins[which] = fwd.make_dual(ins[which], torch.ones_like(ins[which]))
        with pytest.raises(RuntimeError, match="forward"):
            scao_amd.gated_ffn(*ins)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward"):
            scao_amd.gated_ffn(*ins)

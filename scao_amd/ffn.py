"""The gated feed-forward block of a decoder layer, forward and backward.

    y = (f(x Wg^T) * (x Wu^T)) Wd^T

with the weights in ``nn.Linear``'s layout (gate and up: ``d_ff x d_model``, down:
``d_model x d_ff``): the three largest matrices of a layer, whose gradients are
what ``SCAO`` preconditions.  Both projections, the activation and the product
are one kernel, the second projection another; a backward pass is four products
(``scao_ffn_forward``, ``scao_ffn_backward``).  Everything runs on the current
stream; nothing is kept between calls.
"""

from __future__ import annotations

import math

import numpy as np
import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from . import _lib as L
from .engine import require_hip

ACTIVATIONS = {"silu": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3, "sigmoid": 4}


def _check(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, activation: str) -> int:
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)} (got {activation!r})")
    if x.dtype not in L.DTYPE_CODE:
        raise TypeError(f"x must be float32, bfloat16 or float16 (got {x.dtype})")
    for t, name in ((x, "x"), (w_gate, "w_gate"), (w_up, "w_up"), (w_down, "w_down")):
        if not t.is_cuda:
            require_hip(t, name)
        if t.dtype != x.dtype or t.device != x.device:
            raise TypeError(f"{name} is {t.dtype} on {t.device}, x is {x.dtype} on {x.device}")
    if x.ndim < 1 or w_gate.ndim != 2:
        raise ValueError(f"x must have at least one dimension and w_gate two (got "
                         f"{tuple(x.shape)}, {tuple(w_gate.shape)})")
    f, d = w_gate.shape
    if x.shape[-1] != d or w_up.shape != (f, d) or w_down.shape != (d, f):
        raise ValueError(f"shape mismatch: x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up "
                         f"{tuple(w_up.shape)}, w_down {tuple(w_down.shape)}")
    return act


def _rows(t: Tensor) -> Tensor:
    """2-D with unit column stride and rows that do not overlap."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _desc(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, act: int) -> np.ndarray:
    f, d = w_gate.shape
    return np.array([(x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), w_down.data_ptr(),
                      x.stride(0), w_gate.stride(0), w_up.stride(0), w_down.stride(0),
                      x.shape[0], d, f, L.DTYPE_CODE[x.dtype], act)], dtype=L.FFN_DESC)


def _bytes(n: int, device: torch.device) -> Tensor:
    return torch.empty(n, dtype=torch.uint8, device=device)


def _forward(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor, act: int, save: bool):
    """x is 2-D and no size is zero; (y, what the backward pass needs or None)"""
    dev = x.device
    desc = _desc(x, w_gate, w_up, w_down, act)
    at, lib = desc.ctypes.data, L.lib()
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    saved = _bytes(lib.scao_ffn_saved_bytes(at), dev) if save else None
    work = _bytes(lib.scao_ffn_forward_workspace(at, int(save)), dev)
    L.call_on(dev, "scao_ffn_forward", at, y.data_ptr(), saved.data_ptr() if save else None,
              work.data_ptr())
    return y, saved


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, act):
        y, saved = _forward(x, w_gate, w_up, w_down, act, True)
        ctx.save_for_backward(x, w_gate, w_up, w_down, saved)
        ctx.act = act
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        # (hooks on saved tensors may have moved them: their addresses are new)
        x, w_gate, w_up, w_down, saved = ctx.saved_tensors
        dy, dev, dtype = _rows(dy), x.device, x.dtype
        (f, d), need = w_gate.shape, ctx.needs_input_grad
        desc = _desc(x, w_gate, w_up, w_down, ctx.act)
        at = desc.ctypes.data

        def new(want, *shape):
            return torch.empty(shape, dtype=dtype, device=dev) if want else None

        dx, ddown = new(need[0], x.shape[0], d), new(need[3], d, f)
        dgate, dup = new(need[1], f, d), new(need[2], f, d)
        grads = need[0] | need[1] << 1 | need[2] << 2 | need[3] << 3
        dy_at, ld = dy.data_ptr(), dy.stride(0)
        work = _bytes(L.lib().scao_ffn_backward_workspace(at, dy_at, ld, grads), dev)
        L.call_on(dev, "scao_ffn_backward", at, dy_at, ld, saved.data_ptr(),
                  *[None if t is None else t.data_ptr() for t in (dx, dgate, dup, ddown)],
                  work.data_ptr())
        return dx, dgate, dup, ddown, None


def gated_ffn(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor,
              activation: str = "silu") -> Tensor:
    """``(f(x w_gate^T) * (x w_up^T)) w_down^T`` with f one of ``silu``, ``gelu``,
    ``gelu_tanh``, ``relu`` and ``sigmoid``.

    x: ``(..., d_model)``; w_gate, w_up: ``(d_ff, d_model)``; w_down: ``(d_model,
    d_ff)``, all float32, bfloat16 or float16 on one ROCm device.  Rows may have
    any stride (the halves of a packed gate-and-up weight, a slice of a wider
    input) and start at any element; columns of another stride are copied first.
    Sums are float32; the 16-bit types round h, and in the backward pass the
    gradients of both projections, once to the type before the next product.
    Differentiable once, in any of the four arguments."""
    act = _check(x, w_gate, w_up, w_down, activation)
    if x.numel() == 0 or w_gate.numel() == 0:
        # no token, or a sum over nothing: zeros, with gradients that are zeros
        return ((x @ w_gate.t()) * (x @ w_up.t())) @ w_down.t()
    x2, wg, wu, wd = _rows(x), _rows(w_gate), _rows(w_up), _rows(w_down)
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad
                                    or w_down.requires_grad):
        y = _GatedFFN.apply(x2, wg, wu, wd, act)
    else:
        y = _forward(x2, wg, wu, wd, act, False)[0]
    return y if x.dim() == 2 else y.view(x.shape)


class GatedFFN(nn.Module):
    """``gated_ffn`` with its weights: ``gate`` and ``up`` in one parameter
    ``gate_up`` (2 d_ff x d_model, or two with ``packed=False``: ``gate`` and
    ``up``), and ``down`` (d_model x d_ff), initialised as ``nn.Linear`` does."""

    def __init__(self, d_model: int, d_ff: int, activation: str = "silu", packed: bool = False,
                 device=None, dtype=None) -> None:
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)} "
                             f"(got {activation!r})")
        self.d_model, self.d_ff, self.activation, self.packed = d_model, d_ff, activation, packed
        kw = dict(device=device, dtype=dtype)
        if packed:
            self.gate_up = nn.Parameter(torch.empty(2 * d_ff, d_model, **kw))
        else:
            self.gate = nn.Parameter(torch.empty(d_ff, d_model, **kw))
            self.up = nn.Parameter(torch.empty(d_ff, d_model, **kw))
        self.down = nn.Parameter(torch.empty(d_model, d_ff, **kw))
        self.reset_parameters()

    @torch.no_grad()
    def reset_parameters(self) -> None:
        for p in self.parameters():
            bound = 1.0 / math.sqrt(p.shape[1])
            p.uniform_(-bound, bound)

    def forward(self, x: Tensor) -> Tensor:
        gate, up = self.gate_up.split(self.d_ff) if self.packed else (self.gate, self.up)
        return gated_ffn(x, gate, up, self.down, self.activation)

    def extra_repr(self) -> str:
        return f"{self.d_model}, {self.d_ff}, activation={self.activation}, packed={self.packed}"

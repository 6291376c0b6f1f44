"""The gated feed-forward block of a decoder layer, forward and backward.

    y = (f(x Wg^T) * (x Wu^T)) Wd^T

with the weights in ``nn.Linear``'s layout (gate and up: ``d_ff x d_model``, down:
``d_model x d_ff``): the three largest matrices of a layer, whose gradients are
what ``SCAO`` preconditions.  Both projections, the activation and the product
are one kernel, the second projection another; a backward pass is four products
(``scao_ffn_forward``, ``scao_ffn_backward``, called from csrc/torch_host.cpp as
operators of torch's dispatcher).  Everything runs on the current stream; nothing is kept
between calls.
"""

from __future__ import annotations

import math

import torch
from torch import Tensor, nn

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


def gated_ffn(x: Tensor, w_gate: Tensor, w_up: Tensor, w_down: Tensor,
              activation: str = "silu") -> Tensor:
    """``(f(x w_gate^T) * (x w_up^T)) w_down^T`` with f one of ``silu``, ``gelu``,
    ``gelu_tanh``, ``relu`` and ``sigmoid``.

    x: ``(..., d_model)``; w_gate, w_up: ``(d_ff, d_model)``; w_down: ``(d_model,
    d_ff)``, all float32, bfloat16 or float16 on one ROCm device.  Rows may have
    any stride (the halves of a packed gate-and-up weight, a slice of a wider
    input) and start at any element; columns of another stride, and rows 2^21
    elements and more apart, are copied first.  Sums are float32; the 16-bit
    types round h, and in the backward pass the gradients of both projections,
    once to the type before the next product.  Differentiable once, in any of
    the four arguments, not in forward mode."""
    act = _check(x, w_gate, w_up, w_down, activation)
    if x.numel() == 0 or w_gate.numel() == 0:
        # no token, or a sum over nothing: zeros, with gradients that are zeros
        return ((x @ w_gate.t()) * (x @ w_up.t())) @ w_down.t()
    if x.dim() == 2:
        return L.torch_host().gated_ffn(x, w_gate, w_up, w_down, act)
    return L.torch_host().gated_ffn(x.reshape(-1, x.shape[-1]), w_gate, w_up, w_down,
                                    act).view(x.shape)


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
            bound = 1.0 / math.sqrt(p.shape[1]) if p.shape[1] else 0.0
            p.uniform_(-bound, bound)

    def forward(self, x: Tensor) -> Tensor:
        gate, up = self.gate_up.split(self.d_ff) if self.packed else (self.gate, self.up)
        return gated_ffn(x, gate, up, self.down, self.activation)

    def extra_repr(self) -> str:
        return f"{self.d_model}, {self.d_ff}, activation={self.activation}, packed={self.packed}"

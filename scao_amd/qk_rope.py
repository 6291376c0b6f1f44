"""Norms of queries and keys for each head, with the rotation by the token's
position in the same pass, forward and backward.

    y = w x / sqrt(mean(x^2) + eps) over a head's columns, and the pairs of y's first
    columns turned:  y'_i = y_i cos - y_j sin,  y'_j = y_j cos + y_i sin

What a decoder layer does between its projections and the attention: normed heads
bound the attention's logits, which an update that moves all directions of a
projection alike (``Muon``) would otherwise let grow.  Queries and keys go through
one kernel each way (``scao_qk_rope_forward``, ``scao_qk_rope_backward``, called from
csrc/torch_host.cpp as operators of torch's dispatcher) on the current stream; the
backward pass needs nothing but the inputs.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor, nn

from . import _lib as L
from .engine import require_hip

MAX_HEAD_DIM = 512


def rotary_table(length: int, rotary_dim: int, base: float = 10000.0, device=None
                 ) -> Tuple[Tensor, Tensor]:
    """cos and sin of the angles ``p base^(-2 i / rotary_dim)`` of positions p below
    ``length``, i below ``rotary_dim / 2``: float32 tables ``(length, rotary_dim /
    2)``, with the angles in 64 bits."""
    if rotary_dim < 0 or rotary_dim % 2 or length < 0 or not base > 0.0:
        raise ValueError(f"no table of length {length}, rotary_dim {rotary_dim} (even), "
                         f"base {base}")
    half = rotary_dim // 2
    i = torch.arange(half, device=device, dtype=torch.float64)
    angles = torch.arange(length, device=device, dtype=torch.float64)[:, None] * (
        float(base) ** (-i / max(half, 1)))
    return angles.cos().float(), angles.sin().float()


def _check(q: Tensor, k: Tensor, q_weight, k_weight, cos: Tensor, sin: Tensor, positions,
           eps: float) -> None:
    for t, name in ((q, "q"), (k, "k")):
        if not t.is_cuda:
            require_hip(t, name)
        if t.dtype not in L.DTYPE_CODE:
            raise TypeError(f"{name} must be float32, bfloat16 or float16 (got {t.dtype})")
        if t.ndim < 2:
            raise ValueError(f"{name} must be (..., heads, head_dim) (got {tuple(t.shape)})")
    if k.dtype != q.dtype or k.device != q.device:
        raise TypeError(f"k is {k.dtype} on {k.device}, q is {q.dtype} on {q.device}")
    if q.shape[:-2] != k.shape[:-2] or q.shape[-1] != k.shape[-1]:
        raise ValueError(f"shape mismatch: q {tuple(q.shape)}, k {tuple(k.shape)}")
    dim = q.shape[-1]
    if not 1 <= dim <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be from 1 to {MAX_HEAD_DIM} (got {dim})")
    if q.shape[-2] < 1 or k.shape[-2] < 1:
        raise ValueError(f"no heads: q {tuple(q.shape)}, k {tuple(k.shape)}")
    for t, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if t is None:
            continue
        if t.shape != (dim,):
            raise ValueError(f"{name} must be ({dim},) (got {tuple(t.shape)})")
        if t.dtype not in L.DTYPE_CODE or t.device != q.device:
            raise TypeError(f"{name} is {t.dtype} on {t.device}")
    if cos.ndim != 2 or cos.shape != sin.shape or 2 * cos.shape[1] > dim:
        raise ValueError(f"cos and sin must be tables (positions, up to {dim // 2}) of one shape "
                         f"(got {tuple(cos.shape)}, {tuple(sin.shape)})")
    for t, name in ((cos, "cos"), (sin, "sin")):
        if t.dtype != torch.float32 or t.device != q.device:
            raise TypeError(f"{name} must be float32 on {q.device} (got {t.dtype} on {t.device})")
    if positions is not None:
        if positions.dtype not in (torch.int64, torch.int32) or positions.device != q.device:
            raise TypeError("positions must be int64 or int32 on q's device (got "
                            f"{positions.dtype} on {positions.device})")
        if positions.shape != q.shape[:-2]:
            raise ValueError(f"positions must be {tuple(q.shape[:-2])} (got "
                             f"{tuple(positions.shape)})")
    elif q.ndim > 2 and cos.shape[1] and q.shape[-3] > cos.shape[0]:
        raise ValueError(f"{q.shape[-3]} tokens and a table of {cos.shape[0]} positions")
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be at least 0 and finite (got {eps})")


def qk_norm_rope(q: Tensor, k: Tensor, q_weight: Optional[Tensor], k_weight: Optional[Tensor],
                 cos: Tensor, sin: Tensor, positions: Optional[Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False) -> Tuple[Tensor, Tensor]:
    """Both normed for each head and rotated, as fresh tensors of their own types.

    q: ``(..., tokens, q_heads, head_dim)``, k: ``(..., tokens, k_heads, head_dim)``,
    float32, bfloat16 or float16, of any strides (slices of one projection's rows;
    heads before tokens, transposed).  q_weight, k_weight: ``(head_dim,)`` of any of
    the three types, or None for ones.  cos, sin: float32 tables ``(positions,
    rotary_dim / 2)`` (``rotary_table``); the first ``rotary_dim`` columns turn, pairs
    of them half a rotary_dim apart, or side by side with ``interleaved``.
    positions: int64 or int32, one a token, by default a token's place in its
    sequence; one outside of the tables gives NaN in that token's rotated columns.

    Sums and products are float32, every output is rounded once.  Differentiable
    once in q, k and the weights, not in the tables, and not in forward mode.  A head
    with a NaN or an infinity gives NaN there (an infinity: zeros beside it), in its
    gradient and in the weight's, and in no other head; one whose sum of squares is past
    float32's range (values of 1e19) is all zeros, as beside an infinity."""
    rest = q_weight, k_weight, cos, sin
    if q.ndim == 4 and q.is_cuda:
        # the operator checks for itself, in a sixth of the time; what it refuses is
        # looked at again for the error's type and words
        try:
            return L.torch_host().qk_norm_rope(q, k, *rest, positions, eps, interleaved)
        except (RuntimeError, TypeError):
            _check(q, k, *rest, positions, eps)
            raise
    _check(q, k, *rest, positions, eps)
    lead = q.shape[:-2]
    tokens, many = lead[-1] if lead else 1, math.prod(lead[:-1])
    q, k = (t.reshape(many, tokens, *t.shape[-2:]) for t in (q, k))
    if positions is not None:
        positions = positions.reshape(many, tokens)
    yq, yk = L.torch_host().qk_norm_rope(q, k, *rest, positions, eps, interleaved)
    return yq.reshape(*lead, *yq.shape[-2:]), yk.reshape(*lead, *yk.shape[-2:])


class QKNormRope(nn.Module):
    """``qk_norm_rope`` with its weights (``q``, ``k``: ones at first) and the tables
    of ``max_positions`` positions."""

    def __init__(self, head_dim: int, max_positions: int, rotary_dim: Optional[int] = None,
                 base: float = 10000.0, eps: float = 1e-6, interleaved: bool = False, device=None,
                 dtype=None) -> None:
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if not 1 <= head_dim <= MAX_HEAD_DIM or not 0 <= rotary_dim <= head_dim:
            raise ValueError(f"head_dim must be from 1 to {MAX_HEAD_DIM} and rotary_dim at most "
                             f"that (got {head_dim}, {rotary_dim})")
        self.head_dim, self.rotary_dim, self.base = head_dim, rotary_dim, base
        self.eps, self.interleaved = eps, interleaved
        self.q = nn.Parameter(torch.ones(head_dim, device=device, dtype=dtype))
        self.k = nn.Parameter(torch.ones(head_dim, device=device, dtype=dtype))
        cos, sin = rotary_table(max_positions, rotary_dim, base, device)
        self.register_buffer("cos", cos, persistent=False)
        self.register_buffer("sin", sin, persistent=False)

    def _apply(self, fn, *args, **kwargs):
        """(a conversion to another type leaves the tables in 32 bits)"""
        tables = self.cos, self.sin
        super()._apply(fn, *args, **kwargs)
        if self.cos.dtype != torch.float32:
            self.cos, self.sin = (t.to(self.q.device) for t in tables)
        return self

    def forward(self, q: Tensor, k: Tensor, positions: Optional[Tensor] = None
                ) -> Tuple[Tensor, Tensor]:
        return qk_norm_rope(q, k, self.q, self.k, self.cos, self.sin, positions, self.eps,
                            self.interleaved)

    def extra_repr(self) -> str:
        return (f"{self.head_dim}, max_positions={self.cos.shape[0]}, rotary_dim={self.rotary_dim}, "
                f"base={self.base}, interleaved={self.interleaved}")

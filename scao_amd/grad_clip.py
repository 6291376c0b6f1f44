"""Norm over all gradients of a model, and their clipping to it: what a
training loop does between ``loss.backward()`` and ``SCAO.step()``.

    scale = 1 / micro_batches
    norm = scao_amd.clip_grad_norm_(model.parameters(), 1.0, scale=scale)
    opt.step()

The call forms are ``torch.nn.utils.clip_grad_norm_``'s (without ``foreach``),
with ``scale`` for gradients that are a sum of micro-batches or carry a loss
scale: it multiplies every gradient in the same pass.  The gradients of all
tensors go through two kernels (``scao_grad_norm`` / ``scao_grad_clip``, called
from csrc/torch_host.cpp as operators of torch's dispatcher) on the current
stream, without a host synchronisation and without a copy of the tensors' table.
"""

from __future__ import annotations

import math
from typing import Iterable, Union

import torch
from torch import Tensor

from . import _lib as L
from .engine import require_hip

_NORM_CODE = {1.0: 1, 2.0: 2, math.inf: 0}


def _check_scalars(norm_type: float, scale: float) -> int:
    code = _NORM_CODE.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type must be 1, 2 or inf (got {norm_type})")
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite (got {scale})")
    return code


def _checked(parameters: list) -> list:
    """The gradients of a list that _torch_host does not take."""
    grads = [g for p in parameters if (g := p.grad) is not None]
    for g in grads:
        require_hip(g, "gradient")
        if g.device != grads[0].device:
            raise RuntimeError("all gradients must be on one device "
                               f"({g.device} vs {grads[0].device})")
        if g.layout != torch.strided or g.dtype not in L.DTYPE_CODE:
            raise TypeError("gradients must be dense float32, bfloat16 or float16 tensors "
                            f"(got {g.dtype}, {g.layout})")
    return grads


def _as_list(parameters: Union[Tensor, Iterable[Tensor]]) -> list:
    """(an iterator's parameters may live in this list alone)"""
    if isinstance(parameters, Tensor):
        return [parameters]
    return parameters if isinstance(parameters, (list, tuple)) else list(parameters)


def _call(host, operator: str, parameters: list, *scalars) -> Tensor:
    norm = host(parameters, *scalars)
    if norm is False:
        grads = _checked(parameters)
        with torch.no_grad():
            norm = getattr(torch.ops.scao_amd, operator)(grads, *scalars) if grads else None
    return torch.tensor(0.0) if norm is None else norm


def global_grad_norm(parameters: Union[Tensor, Iterable[Tensor]], norm_type: float = 2.0,
                     scale: float = 1.0) -> Tensor:
    """``scale`` times the ``norm_type`` norm (1, 2 or inf) of all gradients of
    ``parameters`` as one vector: a 0-dim float32 tensor on their device
    (summed in double), a zero on the CPU where no parameter has a gradient."""
    code = _check_scalars(norm_type, scale)
    return _call(L.torch_host().grad_norm, "grad_norm", _as_list(parameters), code, float(scale))


def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float,
                    norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    scale: float = 1.0) -> Tensor:
    """Multiply every gradient in place by ``scale * min(1, max_norm / (N +
    1e-6))`` with N = ``global_grad_norm(parameters, norm_type, scale)``, and
    return N (0-dim float32).  Each gradient is rounded once, to its type; with
    a factor of exactly 1 nothing is written.  A NaN in any gradient makes N and
    all gradients NaN, an infinity makes N infinite and the factor 0 (``scale``
    with a max_norm of infinity, which clips nothing), unless
    ``error_if_nonfinite``: then N is read back (the host waits for it) and a
    RuntimeError is raised with the gradients as they were.

    Gradients may have any type of float32, bfloat16 and float16, any start and
    any strides, but no two may share memory (ValueError)."""
    code, max_norm = _check_scalars(norm_type, scale), float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be at least 0 (got {max_norm})")
    parameters, host = _as_list(parameters), L.torch_host()
    if error_if_nonfinite:
        norm = float(_call(host.grad_norm, "grad_norm", parameters, code, float(scale)))
        if not math.isfinite(norm):
            raise RuntimeError(f"the gradients' norm of order {float(norm_type)} is {norm}, so "
                               "they cannot be clipped; pass error_if_nonfinite=False to scale "
                               "them by it anyway")
    return _call(host.grad_clip, "grad_clip_", parameters, code, float(scale), max_norm)

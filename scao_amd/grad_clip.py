"""Norm over all gradients of a model, and their clipping to it: what a
training loop does between ``loss.backward()`` and ``SCAO.step()``.

    scale = 1 / micro_batches
    norm = scao_amd.clip_grad_norm_(model.parameters(), 1.0, scale=scale)
    opt.step()

The call forms are ``torch.nn.utils.clip_grad_norm_``'s, with ``scale`` for
gradients that are a sum of micro-batches or carry a loss scale: it multiplies
every gradient in the same pass.  The gradients of all tensors go through two
kernels (``scao_grad_norm`` / ``scao_grad_clip``) on the current stream, without
a host synchronisation and without a copy of the tensors' table.
"""

from __future__ import annotations

import math
import operator
from typing import Iterable, Union

import numpy as np
import torch
from torch import Tensor

from . import _lib as L
from .engine import require_hip

_NORM_CODE = {1.0: 1, 2.0: 2, math.inf: 0}


def _gradients(parameters: Union[Tensor, Iterable[Tensor]]) -> list:
    if isinstance(parameters, Tensor):
        parameters = [parameters]
    return [g for p in parameters if (g := p.grad) is not None]


# A model has hundreds of gradients, and each attribute of a tensor costs about
# 70 ns of host time: every property is read once, for all of them in one go.
_dtype, _is_sparse = operator.attrgetter("dtype"), operator.attrgetter("is_sparse")


def _check(grads: list, norm_type: float, scale: float) -> tuple:
    """(the norm's code, the gradients' dtype codes, whether all are contiguous)"""
    code = _NORM_CODE.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type must be 1, 2 or inf (got {norm_type})")
    if not 0.0 < scale < math.inf:
        raise ValueError(f"scale must be positive and finite (got {scale})")
    devices = set(map(Tensor.get_device, grads))
    if len(devices) > 1 or -1 in devices:
        for g in grads:
            require_hip(g, "gradient")
        raise RuntimeError(f"all gradients must be on one device (got devices {sorted(devices)})")
    types = list(map(L.DTYPE_CODE.get, map(_dtype, grads)))
    if None in types or any(map(_is_sparse, grads)):
        raise TypeError("gradients must be dense float32, bfloat16 or float16 tensors (got "
                        f"{sorted({f'{g.dtype} {g.layout}' for g in grads})})")
    return code, types, all(map(Tensor.is_contiguous, grads))


def _dense(g: Tensor) -> bool:
    """Every element of the gradient's memory range once, in any order."""
    return g.is_contiguous() or torch.ops.aten.is_non_overlapping_and_dense(g)


def _launch(name: str, grads: list, types: list, code: int, *scalars: float) -> Tensor:
    n = len(grads)
    table = np.empty(n, dtype=L.TENSOR_DESC)
    table["data"] = list(map(Tensor.data_ptr, grads))
    table["numel"] = list(map(Tensor.numel, grads))
    table["dtype"] = types
    at = table.ctypes.data
    dev = grads[0].device
    norm = torch.empty((), dtype=torch.float32, device=dev)
    work = torch.empty(L.lib().scao_grad_norm_workspace(at, n), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        L.call(name, at, n, code, *scalars, norm.data_ptr(), work.data_ptr(), L.stream_ptr(dev))
    return norm


@torch.no_grad()
def global_grad_norm(parameters: Union[Tensor, Iterable[Tensor]], norm_type: float = 2.0,
                     scale: float = 1.0) -> Tensor:
    """``scale`` times the ``norm_type`` norm (1, 2 or inf) of all gradients of
    ``parameters`` as one vector: a 0-dim float32 tensor on their device
    (summed in double), a zero on the CPU where no parameter has a gradient."""
    grads = _gradients(parameters)
    code, types, contiguous = _check(grads, norm_type, scale)
    if not grads:
        return torch.tensor(0.0)
    if not contiguous:
        grads = [g if _dense(g) else g.contiguous() for g in grads]
    return _launch("scao_grad_norm", grads, types, code, float(scale))


@torch.no_grad()
def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float,
                    norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    scale: float = 1.0) -> Tensor:
    """Multiply every gradient in place by ``scale * min(1, max_norm / (N +
    1e-6))`` with N = ``global_grad_norm(parameters, norm_type, scale)``, and
    return N (0-dim float32).  Each gradient is rounded once, to its type; with
    a factor of exactly 1 nothing is written.  A NaN in any gradient makes N and
    all gradients NaN, an infinity makes N infinite and the factor 0, unless
    ``error_if_nonfinite``: then N is read back (the host waits for it) and a
    RuntimeError is raised with the gradients as they were.

    Gradients may have any type of float32, bfloat16 and float16, any start and
    any strides, but no two may share memory (ValueError)."""
    grads = _gradients(parameters)
    code, types, contiguous = _check(grads, norm_type, scale)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be at least 0 (got {max_norm})")
    if not grads:
        return torch.tensor(0.0)
    flat = grads
    if not contiguous:
        flat = [g if _dense(g) else g.contiguous() for g in grads]
        if any(f is not g and torch._debug_has_internal_overlap(g) == 1
               for f, g in zip(flat, grads)):
            raise ValueError("a gradient whose elements share memory (an expanded tensor) "
                             "cannot be scaled in place")
    if error_if_nonfinite:
        norm = float(_launch("scao_grad_norm", flat, types, code, float(scale)))
        if not math.isfinite(norm):
            raise RuntimeError(f"the gradients' norm of order {float(norm_type)} is {norm}, so "
                               "they cannot be clipped; pass error_if_nonfinite=False to scale "
                               "them by it anyway")
    try:
        norm = _launch("scao_grad_clip", flat, types, code, float(scale), max_norm)
    except L.ScaoLibError as e:
        if "share memory" in str(e):
            raise ValueError(str(e)) from None
        raise
    if not contiguous:
        for g, f in zip(grads, flat):
            if f is not g:
                g.copy_(f)
    return norm

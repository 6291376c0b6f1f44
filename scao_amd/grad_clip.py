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

import ctypes
import math
from typing import Iterable, Union

import numpy as np
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


def _irregular(parameters: list) -> list:
    """The gradients of a list that ``_lib.torch_host().gradients`` does not take, checked."""
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


def _dense(g: Tensor) -> bool:
    """Every element of the gradient's memory range once, in any order."""
    return g.is_contiguous() or torch.ops.aten.is_non_overlapping_and_dense(g)


class _Gradients:
    """The table of the parameters' gradients; those with gaps in their memory
    take part through a contiguous copy."""

    def __init__(self, parameters: Union[Tensor, Iterable[Tensor]]):
        if isinstance(parameters, Tensor):
            parameters = [parameters]
        elif not isinstance(parameters, (list, tuple)):
            parameters = list(parameters)
        # until the kernels are queued: an iterator's parameters may live here alone
        self._parameters = parameters
        self.copies = []   # (gradient, its copy)
        found = L.torch_host().gradients(parameters)
        if found is not None:
            index, self.count, self._table = found
            self.device = torch.device("cuda", index) if self.count else None
            self.at = ctypes.cast(self._table, ctypes.c_void_p).value
            return
        grads = _irregular(parameters)
        flat = [g if _dense(g) else g.contiguous() for g in grads]
        self.copies = [(g, f) for g, f in zip(grads, flat) if f is not g]
        self.count, self.device = len(flat), flat[0].device
        self._table = np.empty(self.count, dtype=L.TENSOR_DESC)
        for field, of in (("data", Tensor.data_ptr), ("numel", Tensor.numel),
                          ("dtype", lambda g: L.DTYPE_CODE[g.dtype])):
            self._table[field] = [of(g) for g in flat]
        self.at, self._flat = self._table.ctypes.data, flat

    def launch(self, name: str, code: int, *scalars: float) -> Tensor:
        norm = torch.empty((), dtype=torch.float32, device=self.device)
        work = torch.empty(L.lib().scao_grad_norm_workspace(self.at, self.count),
                           dtype=torch.uint8, device=self.device)
        L.call_on(self.device, name, self.at, self.count, code, *scalars, norm.data_ptr(),
                  work.data_ptr())
        return norm


@torch.no_grad()
def global_grad_norm(parameters: Union[Tensor, Iterable[Tensor]], norm_type: float = 2.0,
                     scale: float = 1.0) -> Tensor:
    """``scale`` times the ``norm_type`` norm (1, 2 or inf) of all gradients of
    ``parameters`` as one vector: a 0-dim float32 tensor on their device
    (summed in double), a zero on the CPU where no parameter has a gradient."""
    code, grads = _check_scalars(norm_type, scale), _Gradients(parameters)
    if not grads.count:
        return torch.tensor(0.0)
    return grads.launch("scao_grad_norm", code, float(scale))


@torch.no_grad()
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
    grads = _Gradients(parameters)
    if not grads.count:
        return torch.tensor(0.0)
    if any(torch._debug_has_internal_overlap(g) == 1 for g, _ in grads.copies):
        raise ValueError("a gradient whose elements share memory (an expanded tensor) cannot be "
                         "scaled in place")
    if error_if_nonfinite:
        norm = float(grads.launch("scao_grad_norm", code, float(scale)))
        if not math.isfinite(norm):
            raise RuntimeError(f"the gradients' norm of order {float(norm_type)} is {norm}, so "
                               "they cannot be clipped; pass error_if_nonfinite=False to scale "
                               "them by it anyway")
    try:
        norm = grads.launch("scao_grad_clip", code, float(scale), max_norm)
    except L.ScaoLibError as e:
        if "share memory" in str(e):
            raise ValueError(str(e)) from None
        raise
    for g, copy in grads.copies:
        g.copy_(copy)
    return norm

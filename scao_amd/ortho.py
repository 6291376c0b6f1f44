"""Matrix updates made orthogonal by Newton-Schulz products, and the optimiser
that is built on them.

    X = G / (|G| + eps);  A = X X^T;  X <- a X + (b A + c A A) X,  a few times

on a matrix's smaller side sends its singular values through the polynomials a s
+ b s^3 + c s^5 and leaves its singular vectors: an update whose directions all
have about the same size.  All matrices of a call, whatever their shapes, go
through the same launches (``scao_orthogonalize``, ``scao_muon_step``, called from
csrc/torch_host.cpp as operators of torch's dispatcher) on the current stream;
nothing is kept between calls.
"""

from __future__ import annotations

import math
from typing import Iterable, Optional, Sequence, Union

import torch
from torch import Tensor

from . import _lib as L
from .engine import require_hip

NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _flat_coefficients(coefficients, steps: int) -> list:
    """Three numbers a step."""
    if not isinstance(steps, int) or isinstance(steps, bool) or not 1 <= steps <= 64:
        raise ValueError(f"steps must be a whole number from 1 to 64 (got {steps!r})")
    rows = list(coefficients)
    if rows and not isinstance(rows[0], (list, tuple)):
        rows = [rows] * steps
    if len(rows) != steps or any(len(r) != 3 for r in rows):
        raise ValueError("coefficients must be three numbers, or three of every step "
                         f"(got {coefficients!r} for {steps} steps)")
    flat = [float(x) for r in rows for x in r]
    if not all(map(math.isfinite, flat)):
        raise ValueError(f"coefficients must be finite (got {coefficients!r})")
    return flat


def _check_eps(eps: float) -> float:
    eps = float(eps)
    if not 1e-300 <= eps < math.inf:
        raise ValueError(f"eps must be finite and at least 1e-300 (got {eps})")
    return eps


def _check_ns_dtype(ns_dtype) -> None:
    if ns_dtype not in (None, torch.float32, torch.bfloat16):
        raise ValueError(f"ns_dtype must be None, torch.float32 or torch.bfloat16 (got {ns_dtype})")


def orthogonalize(updates: Union[Tensor, Sequence[Tensor]], steps: int = 5,
                  coefficients=NS_COEFFICIENTS, eps: float = 1e-7,
                  dtype: Optional[torch.dtype] = None, ns_dtype: Optional[torch.dtype] = None
                  ) -> Union[Tensor, list]:
    """The matrices of ``updates`` with their singular values taken through
    ``steps`` Newton-Schulz steps, as fresh contiguous tensors.

    updates: a matrix or a stack of matrices ``(..., m, n)``, or a list of them,
    of any shapes; float32, bfloat16 or float16 on one ROCm device, rows of any
    stride.  coefficients: (a, b, c), or one such triple a step.  dtype: the
    results' type, that of each update by default.

    ns_dtype: how exact the products are.  torch.bfloat16: of fp16 words (three bits
    more than bfloat16's own), sums in float32; with the defaults 0.6e-3 to 1.4e-3 off,
    where a bfloat16's last rounding is 1.7e-3.  torch.float32: of 22-bit words, at a
    third of the rate (1e-6 to 2e-6 off); matrices of up to 128 rows or columns have
    them in any case.  None: bfloat16 for results of that type, else float32.

    A matrix with a NaN or an infinity gives NaN throughout and no other matrix; one of
    zeros gives zeros.  Coefficients with which a singular value may grow beyond 1024 are
    refused.  eps is meant to be small beside the norms: G / (|G| + eps) is held to 2^-39
    absolutely, whatever the precision.  No derivative."""
    flat, eps = _flat_coefficients(coefficients, steps), _check_eps(eps)
    single = isinstance(updates, Tensor)
    updates = [updates] if single else list(updates)
    for t in updates:
        if not isinstance(t, Tensor):
            raise TypeError(f"updates must be tensors (got {type(t).__name__})")
        if t.ndim < 2:
            raise ValueError(f"updates must be matrices or stacks of them (got {tuple(t.shape)})")
        if not t.is_cuda:
            require_hip(t, "update")
        if t.dtype not in L.DTYPE_CODE or t.layout != torch.strided:
            raise TypeError("updates must be dense float32, bfloat16 or float16 tensors (got "
                            f"{t.dtype}, {t.layout})")
        if t.device != updates[0].device:
            raise RuntimeError(f"updates on {updates[0].device} and {t.device}")
    if dtype is not None and dtype not in L.DTYPE_CODE:
        raise TypeError(f"dtype must be float32, bfloat16 or float16 (got {dtype})")
    _check_ns_dtype(ns_dtype)
    if not updates:
        return []
    L.torch_host()
    out = torch.ops.scao_amd.orthogonalize(updates, flat, eps, dtype, ns_dtype)
    return out[0] if single else out


class Muon(torch.optim.Optimizer):
    """Momentum, orthogonalised, for the matrices of a model:

        m <- mu m + (1 - mu) g;   u = mu m + (1 - mu) g  (nesterov; else m)
        p <- (1 - lr weight_decay) p - lr r orthogonalize(u)

    with r = sqrt(max(1, rows / cols)) (``adjust_lr_fn`` None or "original") or
    0.2 sqrt(max(rows, cols)) ("match_rms_adamw").  The arguments and the state's
    ``momentum_buffer`` are those of ``torch.optim.Muon``; the buffer is float32
    whatever the parameter's type is.  Parameters are contiguous matrices, or
    stacks of them with the matrices last (a convolution's weight would be a stack of its
    kernels: flatten it to a matrix before); vectors and embeddings belong to
    another optimizer, such as ``SCAO``.  One call steps all parameters.  A step can be
    captured into a graph once a step before it has made the momentum.

    ns_dtype: how exact the orthogonalised update is (``orthogonalize``):
    torch.float32, torch.bfloat16, or None: float32 for float32 parameters."""

    def __init__(self, params: Iterable, lr: float = 1e-3, weight_decay: float = 0.1,
                 momentum: float = 0.95, nesterov: bool = True, ns_coefficients=NS_COEFFICIENTS,
                 eps: float = 1e-7, ns_steps: int = 5, adjust_lr_fn: Optional[str] = None,
                 ns_dtype: Optional[torch.dtype] = None) -> None:
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum,
                                      nesterov=nesterov, ns_coefficients=ns_coefficients, eps=eps,
                                      ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn,
                                      ns_dtype=ns_dtype))

    def add_param_group(self, param_group: dict) -> None:
        super().add_param_group(param_group)
        try:
            self._check(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    @staticmethod
    def _check(group: dict) -> list:
        """A group's values as they are now; its coefficients, three a step."""
        if not 0.0 <= group["lr"] < math.inf:
            raise ValueError(f"lr must be at least 0 and finite (got {group['lr']})")
        if not 0.0 <= group["weight_decay"] < math.inf:
            raise ValueError(f"weight_decay must be at least 0 and finite "
                             f"(got {group['weight_decay']})")
        if not 0.0 <= group["momentum"] < 1.0:
            raise ValueError(f"momentum must be in [0, 1) (got {group['momentum']})")
        if group["adjust_lr_fn"] not in (None, "original", "match_rms_adamw"):
            raise ValueError('adjust_lr_fn must be None, "original" or "match_rms_adamw" '
                             f"(got {group['adjust_lr_fn']!r})")
        _check_ns_dtype(group["ns_dtype"])
        _check_eps(group["eps"])
        for p in group["params"]:
            if p.ndim < 2:
                raise ValueError("Muon takes matrices and stacks of them; a parameter has shape "
                                 f"{tuple(p.shape)}")
            if p.dtype not in L.DTYPE_CODE or p.layout != torch.strided:
                raise TypeError("Muon takes dense float32, bfloat16 or float16 parameters (got "
                                f"{p.dtype}, {p.layout})")
        return _flat_coefficients(group["ns_coefficients"], group["ns_steps"])

    def _momentum(self, p: Tensor) -> Tensor:
        state = self.state[p]
        buf = state.get("momentum_buffer")
        ready = buf is not None and buf.dtype == torch.float32 and buf.is_contiguous()
        if not ready and torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            # every replay would start again from the momentum as it is made here
            raise RuntimeError("Muon's first step, which makes the momentum, cannot be captured: "
                               "take one before the capture")
        if buf is None:
            buf = state["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32,
                                                         device=p.device)
        elif not ready:   # another optimizer's state
            buf = state["momentum_buffer"] = buf.to(torch.float32).contiguous()
        return buf

    def __setstate__(self, state: dict) -> None:
        """(the groups of torch.optim.Muon know no ns_dtype)"""
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("ns_dtype", self.defaults["ns_dtype"])

    def load_state_dict(self, state_dict: dict) -> None:
        """(torch's own would round the momentum to the parameter's type.)"""
        super().load_state_dict(state_dict)
        given = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(given, params):
            buf = state_dict["state"].get(i, {}).get("momentum_buffer")
            if buf is not None:
                self.state[p]["momentum_buffer"] = buf.to(
                    device=p.device, dtype=torch.float32, copy=True).contiguous()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        host = L.torch_host()
        queue = []   # what is refused here is refused before any group's step
        for group in self.param_groups:
            flat = self._check(group)
            lr, wd = float(group["lr"]), float(group["weight_decay"])
            calls: dict = {}   # by device
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if not p.is_cuda:
                    require_hip(p, "parameter")
                if g.layout != torch.strided or g.dtype not in L.DTYPE_CODE:
                    raise TypeError("gradients must be dense float32, bfloat16 or float16 tensors "
                                    f"(got {g.dtype}, {g.layout})")
                if not p.is_contiguous():
                    raise ValueError("Muon takes contiguous parameters; one has strides "
                                     f"{p.stride()}")
                if p.numel() == 0:
                    continue
                rows, cols = p.shape[-2:]
                ratio = (0.2 * math.sqrt(max(rows, cols))
                         if group["adjust_lr_fn"] == "match_rms_adamw"
                         else math.sqrt(max(1.0, rows / cols)))
                precise = (group["ns_dtype"] or p.dtype) == torch.float32
                lists = calls.setdefault(p.device, ([], [], [], [], [], []))
                for to, x in zip(lists, (p, g, self._momentum(p), lr * ratio, 1.0 - lr * wd,
                                         L.ORTHO_FP32 if precise else L.ORTHO_FAST)):
                    to.append(x)
            queue += [(*lists, float(group["momentum"]), bool(group["nesterov"]), flat,
                       float(group["eps"]), precisions) for *lists, precisions in calls.values()]
        for call in queue:
            host.muon_step(*call)
        return loss

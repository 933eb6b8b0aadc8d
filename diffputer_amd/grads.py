"""Global norm of many gradient tensors and clipping by it, on the HIP kernels (`dp_grad_norm`, `dp_clip_grads`,
include/diffputer.h): what stands between `mstep.NativeTrainStep.loss_and_grads` and the optimiser's step when the M-step
trains with a limit on the gradient (`em.m_step(max_grad_norm=...)`).

Two passes over memory whatever the number of tensors (one table of pointers per 160 of them, in the kernel's arguments),
sums in float64, no copy to the host.  There is no CPU fallback: for CPU tensors use torch.nn.utils.clip_grad_norm_.
"""
from __future__ import annotations

import math

import torch

from . import _lib

_DTYPES = (torch.float32, torch.bfloat16)
_NORMS = {2.0: _lib.DP_NORM_L2, math.inf: _lib.DP_NORM_MAX}


def _list(grads):
    return [grads] if isinstance(grads, torch.Tensor) else list(grads)


def _kind(norm_type):
    kind = _NORMS.get(float(norm_type))
    if kind is None:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    return kind


def _refuse(grads, what):
    """The error of a list that the kernels do not take."""
    if not grads:
        raise ValueError(f"{what}: no tensors")
    dev = grads[0].device
    for i, g in enumerate(grads):
        if g.dtype not in _DTYPES:
            raise ValueError(f"{what}: tensor {i} is {g.dtype}: float32 and bfloat16 are supported")
        if g.device != dev:
            raise ValueError(f"{what}: tensor {i} is on {g.device}, tensor 0 on {dev}")
    if dev.type != "cuda":
        raise _lib.DiffputerError(f"{what} needs tensors on a CUDA (ROCm) device; there is no CPU fallback")
    raise ValueError(f"{what} takes dense (strided) tensors")


def _call(grads, kind, limit, what):
    """The norm; `grads` are clipped in place if there is a limit."""
    call = _lib.torch_side().grads
    norm = call(grads, kind, limit)
    if norm is None:
        _refuse(grads, what)
    if isinstance(norm, int):                                    # tensor number `norm` does not fill one range of memory: copies
        flat = []
        with torch.no_grad():
            for i, g in enumerate(grads):
                if limit is not None and any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
                    raise ValueError(f"{what}: tensor {i} is expanded: its elements share memory")
                flat.append(g if i < norm or g.is_contiguous() else g.contiguous())
            norm = call(flat, kind, limit)
            if not isinstance(norm, torch.Tensor):
                _refuse(grads, what)
            if limit is not None:
                for g, f in zip(grads, flat):
                    if f is not g:
                        g.copy_(f)
    return norm


def grad_norm(grads, norm_type: float = 2.0) -> torch.Tensor:
    """Norm of all elements of `grads` (a tensor, or an iterable of them: float32 / bfloat16, one device) as a 0-dim float32
    tensor on that device; norm_type 2 or inf.  NaN and infinities propagate.  The norm itself has no derivatives (a tensor with
    a forward-mode tangent is refused)."""
    return _call(_list(grads), _kind(norm_type), None, "grad_norm")


def clip_grads(grads, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales `grads` in place by min(1, max_norm / (norm + 1e-6)) and returns their norm from before (0-dim float32 tensor on
    their device; nothing waits for the GPU).  The rule of torch.nn.utils.clip_grad_norm_, on gradients instead of
    parameters: `clip_grads([p.grad for p in params if p.grad is not None], 1.0)`.

    float32 and bfloat16 mix freely; every tensor has to own its elements once (an expanded tensor, or two that share
    memory, are refused).  error_if_nonfinite: wait for the norm, and raise RuntimeError before anything is scaled if it is
    NaN or infinite (not inside a graph capture)."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm has to be a number of at least 0, got {max_norm}")
    grads, kind = _list(grads), _kind(norm_type)
    if error_if_nonfinite:
        norm = float(_call(grads, kind, None, "clip_grads"))
        if not math.isfinite(norm):
            raise RuntimeError(f"clip_grads: the gradients' norm is {norm}; nothing was scaled")
    return _call(grads, kind, max_norm, "clip_grads")


__all__ = ["grad_norm", "clip_grads"]

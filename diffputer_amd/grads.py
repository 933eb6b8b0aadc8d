"""Global norm of many gradient tensors and clipping by it, on the HIP kernels (`dp_grad_norm`, `dp_clip_grads`,
include/diffputer.h): what stands between `mstep.NativeTrainStep.loss_and_grads` and the optimiser's step when the M-step
trains with a limit on the gradient (`em.m_step(max_grad_norm=...)`).

Two passes over memory whatever the number of tensors (one table of pointers per 160 of them, in the kernel's arguments),
sums in float64, no copy to the host.  There is no CPU fallback: for CPU tensors use torch.nn.utils.clip_grad_norm_.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.DP_DTYPE_F32, torch.bfloat16: _lib.DP_DTYPE_BF16}
_NORMS = {2.0: _lib.DP_NORM_L2, math.inf: _lib.DP_NORM_MAX}


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill one range of memory, each place once (in any order of its dimensions)."""
    if t.is_contiguous():
        return True
    size = 1
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != size:
            return False
        size *= n
    return True


def _check(grads, norm_type, what):
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    if float(norm_type) not in _NORMS:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
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
    return grads, dev


def _call(name, grads, norm_type, dev, limit=None):
    lib = _lib.load()
    n = len(grads)
    ptrs = (C.c_void_p * n)(*[g.data_ptr() for g in grads])
    numel = (C.c_int64 * n)(*[g.numel() for g in grads])
    dtypes = (C.c_int * n)(*[_DTYPES[g.dtype] for g in grads])
    with torch.cuda.device(dev):
        norm = torch.empty((), dtype=torch.float32, device=dev)
        ws = torch.empty(lib.dp_grad_workspace_bytes(n), dtype=torch.uint8, device=dev)
        rest = (norm.data_ptr(), ws.data_ptr(), ws.numel(), C.c_void_p(torch.cuda.current_stream(dev).cuda_stream))
        args = (n, ptrs, numel, dtypes, _NORMS[float(norm_type)])
        rc = getattr(lib, name)(*args, *rest) if limit is None else getattr(lib, name)(*args, limit, *rest)
    _lib.check(rc, name)
    return norm


def grad_norm(grads, norm_type: float = 2.0) -> torch.Tensor:
    """Norm of all elements of `grads` (a tensor, or an iterable of them: float32 / bfloat16, one device) as a 0-dim float32
    tensor on that device; norm_type 2 or inf.  NaN and infinities propagate."""
    grads, dev = _check(grads, norm_type, "grad_norm")
    with torch.no_grad():
        return _call("dp_grad_norm", [g if _dense(g) else g.contiguous() for g in grads], norm_type, dev)


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
    grads, dev = _check(grads, norm_type, "clip_grads")
    with torch.no_grad():
        flat = []
        for i, g in enumerate(grads):
            if _dense(g):
                flat.append(g)
            elif any(s == 0 and n > 1 for s, n in zip(g.stride(), g.shape)):
                raise ValueError(f"clip_grads: tensor {i} is expanded: its elements share memory")
            else:
                flat.append(g.contiguous())                      # strided: scaled as a copy and written back
        if error_if_nonfinite:
            norm = _call("dp_grad_norm", flat, norm_type, dev)
            if not math.isfinite(float(norm)):
                raise RuntimeError(f"clip_grads: the gradients' norm is {float(norm)}; nothing was scaled")
        norm = _call("dp_clip_grads", flat, norm_type, dev, max_norm)
        for g, f in zip(grads, flat):
            if f is not g:
                g.copy_(f)
    return norm


__all__ = ["grad_norm", "clip_grads"]

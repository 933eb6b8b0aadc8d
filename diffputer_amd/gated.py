"""Gated projection on the HIP kernels: `h = act(x Wg^T + bg) * (x Wu^T + bu)` (`dp_gated_linear`, include/diffputer.h).

The gated counterpart of `sampler.linear` (act(A W^T + bias)) and of the Linear + SiLU pairs of `model.MLPDiffusion`, for
denoisers built from gated layers: both products, the activation and the gating are one kernel, few rows (a request of one)
have a form of their own, and autograd gets the gradients of x, both weights and both biases from `dp_gated_linear_bwd`.

float32 or bfloat16 throughout; sums, the saved projections and the bias gradients' sums are float32.  There is no CPU
fallback in `gated_linear`; `GatedLinear` computes the same expression in PyTorch where its input is on the CPU, as the
other modules of a denoiser do.
"""
from __future__ import annotations

import ctypes as C
import math

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.DP_DTYPE_F32, torch.bfloat16: _lib.DP_DTYPE_BF16}
_ACTS = {"none": 0, "silu": 1, "gelu": 2}


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[rows, cols] with contiguous rows that do not overlap: `t` itself, or a copy."""
    if t.shape[0] == 0 or ((t.stride(1) == 1 or t.shape[1] == 1) and (t.stride(0) >= t.shape[1] or t.shape[0] == 1)):
        return t
    return t.contiguous()


def _ld(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])                       # a single row's stride says nothing


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(lib, operands, M, N, K, backward, device):
    need = lib.dp_gated_linear_workspace_bytes(*operands, M, N, K, backward)
    if need == 0:
        _lib.check(-1, "dp_gated_linear_workspace_bytes")
    return torch.empty(need, dtype=torch.uint8, device=device)


def _operands(x, w_gate, w_up):
    return _DTYPES[x.dtype], x.data_ptr(), _ld(x), w_gate.data_ptr(), w_up.data_ptr(), _ld(w_gate)


def _stream(device):
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _weights(w_gate, w_up):
    """Both weights with one row stride."""
    w_gate, w_up = _rows(w_gate), _rows(w_up)
    if w_gate.shape[0] > 1 and w_gate.stride(0) != w_up.stride(0):
        w_gate, w_up = w_gate.contiguous(), w_up.contiguous()
    return w_gate, w_up


def _forward(x, w_gate, w_up, b_gate, b_up, act, save):
    lib = _lib.load()
    (M, K), N = x.shape, w_gate.shape[0]
    h = torch.empty((M, N), dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        pre = None
        if save:
            pre = torch.empty(lib.dp_gated_linear_pre_bytes(M, N), dtype=torch.uint8, device=x.device)
        if M:
            ops = _operands(x, w_gate, w_up)
            ws = _workspace(lib, ops, M, N, K, 0, x.device)
            rc = lib.dp_gated_linear(*ops, _ptr(b_gate), _ptr(b_up),
                                     h.data_ptr(), N, _ptr(pre), M, N, K, act, ws.data_ptr(), ws.numel(), _stream(x.device))
            _lib.check(rc, "dp_gated_linear")
    return h, pre


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        w_gate, w_up = _weights(w_gate, w_up)
        h, pre = _forward(x, w_gate, w_up, b_gate, b_up, act, True)
        ctx.save_for_backward(x, w_gate, w_up, pre)
        ctx.act = act
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        lib = _lib.load()
        (M, K), N = x.shape, w_gate.shape[0]
        dh = _rows(dh)

        def out(wanted, *shape):
            return torch.empty(shape, dtype=x.dtype, device=x.device) if wanted else None

        dx = out(need[0], M, K)
        dwg, dwu = out(need[1], N, K), out(need[2], N, K)
        dbg, dbu = out(need[3], N), out(need[4], N)
        with torch.cuda.device(x.device):
            ops = _operands(x, w_gate, w_up)
            ws = _workspace(lib, ops, M, N, K, 1, x.device)
            rc = lib.dp_gated_linear_bwd(*ops, pre.data_ptr(), dh.data_ptr(), _ld(dh),
                                         _ptr(dx), _ptr(dwg), _ptr(dwu), _ptr(dbg), _ptr(dbu), M, N, K, ctx.act, ws.data_ptr(), ws.numel(), _stream(x.device))
        _lib.check(rc, "dp_gated_linear_bwd")
        return dx, dwg, dwu, dbg, dbu, None


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: torch.Tensor | None = None,
                 b_up: torch.Tensor | None = None, act: str = "silu") -> torch.Tensor:
    """act(x @ w_gate^T + b_gate) * (x @ w_up^T + b_up) -> [..., N].

    x [..., K]; w_gate, w_up [N, K]; b_gate, b_up [N] or None each; all of one dtype (float32 or bfloat16) on one CUDA (ROCm)
    device.  act: "silu", "gelu" (g Phi(g), not its tanh approximation) or "none".  Row strides are used as they are (a column range
    of a wider table is not copied); other layouts are copied.  Runs on torch's current stream of x's device; first
    derivatives only.  A row's result does not depend on the rows beside it."""
    if act not in _ACTS:
        raise ValueError(f"act must be one of {sorted(_ACTS)}, got {act!r}")
    if x.ndim < 1 or w_gate.ndim != 2 or w_up.shape != w_gate.shape or x.shape[-1] != w_gate.shape[1]:
        raise ValueError(f"x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)}: expected [..., K], [N, K], [N, K]")
    N, K = w_gate.shape
    if N < 1 or K < 1:
        raise ValueError(f"w_gate {tuple(w_gate.shape)}: N and K have to be at least 1")
    given = [("x", x), ("w_gate", w_gate), ("w_up", w_up), ("b_gate", b_gate), ("b_up", b_up)]
    for name, t in given:
        if t is None:
            continue
        if name.startswith("b_") and tuple(t.shape) != (N,):
            raise ValueError(f"{name} {tuple(t.shape)} does not match N = {N}")
        if t.dtype != x.dtype or t.dtype not in _DTYPES:
            raise ValueError(f"{name} is {t.dtype}: all tensors have to be float32, or all bfloat16")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    if not x.is_cuda:
        raise _lib.DiffputerError("gated_linear needs tensors on a CUDA (ROCm) device; there is no CPU fallback")
    x2 = _rows(x.reshape(math.prod(x.shape[:-1]), K))
    b_gate, b_up = (None if b is None else b.contiguous() for b in (b_gate, b_up))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for _, t in given):
        h = _GatedLinear.apply(x2, w_gate, w_up, b_gate, b_up, _ACTS[act])
    else:
        h = _forward(x2, *_weights(w_gate, w_up), b_gate, b_up, _ACTS[act], False)[0]
    return h.reshape(*x.shape[:-1], N)


class GatedLinear(nn.Module):
    """`act(gate(x)) * up(x)` with `gate`, `up` two Linear layers in_features -> out_features: a gated layer for denoisers that
    `model.Precond` / `model.Model` take as `denoise_fn`.  State-dict keys `gate.weight`, `gate.bias`, `up.weight`, `up.bias`."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, act: str = "silu"):
        super().__init__()
        if act not in _ACTS:
            raise ValueError(f"act must be one of {sorted(_ACTS)}, got {act!r}")
        self.gate = nn.Linear(in_features, out_features, bias=bias)
        self.up = nn.Linear(in_features, out_features, bias=bias)
        self.act = act

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.is_cuda:
            return gated_linear(x, self.gate.weight, self.up.weight, self.gate.bias, self.up.bias, act=self.act)
        g = self.gate(x)
        g = nn.functional.silu(g) if self.act == "silu" else nn.functional.gelu(g) if self.act == "gelu" else g
        return g * self.up(x)

    def extra_repr(self) -> str:
        return f"act={self.act}"


__all__ = ["gated_linear", "GatedLinear"]

"""Gated projection on the HIP kernels: `h = act(x Wg^T + bg) * (x Wu^T + bu)` (`dp_gated_linear`, include/diffputer.h).

The gated counterpart of `sampler.linear` (act(A W^T + bias)) and of the Linear + SiLU pairs of `model.MLPDiffusion`, for
denoisers built from gated layers: both products, the activation and the gating are one kernel, few rows (a request of one)
have a form of their own, and autograd gets the gradients of x, both weights and both biases from `dp_gated_linear_bwd`.

float32 or bfloat16 throughout; sums, the saved projections and the bias gradients' sums are float32.  There is no CPU
fallback in `gated_linear`; `GatedLinear` computes the same expression in PyTorch where its input is on the CPU, as the
other modules of a denoiser do.
"""
from __future__ import annotations

import contextlib
import functools
import math

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.DP_DTYPE_F32, torch.bfloat16: _lib.DP_DTYPE_BF16}
_ACTS = {"none": 0, "silu": 1, "gelu": 2}
_EWORKSPACE = -4


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[rows, cols] with contiguous rows that do not overlap: `t` itself, or a copy."""
    if t.is_contiguous() or t.shape[0] == 0 or ((t.stride(1) == 1 or t.shape[1] == 1) and (t.stride(0) >= t.shape[1] or t.shape[0] == 1)):
        return t
    return t.contiguous()


def _ld(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])                       # a single row's stride says nothing


def _ptr(t):
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=4096)
def _need(dtype, ox, ldx, og, ou, ldw, M, N, K, backward):
    """Workspace bytes of a call: by its sizes, strides and the pointers' alignment (their last 4 bits), nothing else."""
    lib = _lib.load()
    need = lib.dp_gated_linear_workspace_bytes(dtype, 16 + ox, ldx, 16 + og, 16 + ou, ldw, M, N, K, backward)
    if need == 0:
        _lib.check(-1, "dp_gated_linear_workspace_bytes")
    return need


def _call(name, x, w_gate, w_up, rest, M, N, K, act, backward):
    """One call of the C entry `name` on the current stream of x's device, with a workspace of its own."""
    lib = _lib.load()
    dt, px, pg, pu, ldx, ldw = _DTYPES[x.dtype], x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), _ld(x), _ld(w_gate)
    index = x.device.index
    key = (dt, px & 15, ldx, pg & 15, pu & 15, ldw, M, N, K, backward)
    guard = torch.cuda.device(index) if torch.cuda.current_device() != index else contextlib.nullcontext()
    with guard:
        for attempt in range(2):
            need = _need(*key)
            ws = torch.empty(need, dtype=torch.uint8, device=x.device)
            rc = getattr(lib, name)(dt, px, ldx, pg, pu, ldw, *rest, M, N, K, act, ws.data_ptr(), need, torch.cuda.current_stream(index).cuda_stream)
            if rc != _EWORKSPACE or attempt:
                break
            _need.cache_clear()                               # a dp_tune setting changed what the kernels need
    if rc != 0:
        _lib.check(rc, name)


def _forward(x, w_gate, w_up, b_gate, b_up, act, save):
    (M, K), N = x.shape, w_gate.shape[0]
    h = x.new_empty((M, N))
    pre = None
    if save:
        pre = torch.empty(_lib.load().dp_gated_linear_pre_bytes(M, N), dtype=torch.uint8, device=x.device)
    if M:
        _call("dp_gated_linear", x, w_gate, w_up, (_ptr(b_gate), _ptr(b_up), h.data_ptr(), N, _ptr(pre)), M, N, K, act, 0)
    return h, pre


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        h, pre = _forward(x, w_gate, w_up, b_gate, b_up, act, True)
        ctx.save_for_backward(x, w_gate, w_up, pre)
        ctx.act = act
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, pre = ctx.saved_tensors
        need = ctx.needs_input_grad
        (M, K), N = x.shape, w_gate.shape[0]
        dh = _rows(dh)
        dx = x.new_empty((M, K)) if need[0] else None
        dwg = x.new_empty((N, K)) if need[1] else None
        dwu = x.new_empty((N, K)) if need[2] else None
        dbg = x.new_empty(N) if need[3] else None
        dbu = x.new_empty(N) if need[4] else None
        _call("dp_gated_linear_bwd", x, w_gate, w_up, (pre.data_ptr(), dh.data_ptr(), _ld(dh), _ptr(dx), _ptr(dwg), _ptr(dwu), _ptr(dbg), _ptr(dbu)), M, N, K, ctx.act, 1)
        return dx, dwg, dwu, dbg, dbu, None


def _refuse(x, w_gate, w_up, b_gate, b_up, act):
    """The error of a call that gated_linear does not take."""
    if act not in _ACTS:
        raise ValueError(f"act must be one of {sorted(_ACTS)}, got {act!r}")
    if x.ndim < 1 or w_gate.ndim != 2 or w_up.shape != w_gate.shape or x.shape[-1] != w_gate.shape[1]:
        raise ValueError(f"x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)}: expected [..., K], [N, K], [N, K]")
    N, K = w_gate.shape
    if N < 1 or K < 1:
        raise ValueError(f"w_gate {tuple(w_gate.shape)}: N and K have to be at least 1")
    for name, t in (("x", x), ("w_gate", w_gate), ("w_up", w_up), ("b_gate", b_gate), ("b_up", b_up)):
        if t is None:
            continue
        if name.startswith("b_") and tuple(t.shape) != (N,):
            raise ValueError(f"{name} {tuple(t.shape)} does not match N = {N}")
        if t.dtype != x.dtype or t.dtype not in _DTYPES:
            raise ValueError(f"{name} is {t.dtype}: all tensors have to be float32, or all bfloat16")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    raise _lib.DiffputerError("gated_linear needs tensors on a CUDA (ROCm) device; there is no CPU fallback")


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: torch.Tensor | None = None,
                 b_up: torch.Tensor | None = None, act: str = "silu") -> torch.Tensor:
    """act(x @ w_gate^T + b_gate) * (x @ w_up^T + b_up) -> [..., N].

    x [..., K]; w_gate, w_up [N, K]; b_gate, b_up [N] or None each; all of one dtype (float32 or bfloat16) on one CUDA (ROCm)
    device.  act: "silu", "gelu" (g Phi(g), not its tanh approximation) or "none".  Row strides are used as they are (a column range
    of a wider table is not copied); other layouts are copied.  Runs on torch's current stream of x's device; first
    derivatives only.  A row of h depends on its own row of x only."""
    code, dt, dev, shape = _ACTS.get(act), x.dtype, x.device, w_gate.shape
    ok = code is not None and x.is_cuda and dt in _DTYPES and len(shape) == 2 and w_up.shape == shape and x.ndim >= 1 and x.shape[-1] == shape[1] and shape.numel() > 0
    grad = x.requires_grad
    if ok:
        for t in (w_gate, w_up):
            ok = ok and t.dtype == dt and t.device == dev
            grad = grad or t.requires_grad
        for t in (b_gate, b_up):
            if t is not None:
                ok = ok and t.dtype == dt and t.device == dev and t.ndim == 1 and t.shape[0] == shape[0]
                grad = grad or t.requires_grad
    if not ok:
        _refuse(x, w_gate, w_up, b_gate, b_up, act)
    x2 = _rows(x if x.ndim == 2 else x.reshape(math.prod(x.shape[:-1]), shape[1]))
    w_gate, w_up = _rows(w_gate), _rows(w_up)
    if shape[0] > 1 and w_gate.stride(0) != w_up.stride(0):   # the kernels take both weights with one row stride
        w_gate, w_up = w_gate.contiguous(), w_up.contiguous()
    if b_gate is not None and not b_gate.is_contiguous():
        b_gate = b_gate.contiguous()
    if b_up is not None and not b_up.is_contiguous():
        b_up = b_up.contiguous()
    if grad and torch.is_grad_enabled():
        h = _GatedLinear.apply(x2, w_gate, w_up, b_gate, b_up, code)
    else:
        h = _forward(x2, w_gate, w_up, b_gate, b_up, code, False)[0]
    return h if x.ndim == 2 else h.reshape(*x.shape[:-1], shape[0])


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

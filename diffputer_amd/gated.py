"""Gated projection on the HIP kernels: `h = act(x Wg^T + bg) * (x Wu^T + bu)` (`dp_gated_linear`, include/diffputer.h).

The gated counterpart of `sampler.linear` (act(A W^T + bias)) and of the Linear + SiLU pairs of `model.MLPDiffusion`, for
denoisers built from gated layers, which train inside `model.Model` (`em.m_step`, `em.run_em` and the sampler's plans run MLPDiffusion
only): both products, the activation and the gating are one kernel, few rows (a request of one)
have a form of their own, and autograd gets the gradients of x, both weights and both biases from `dp_gated_linear_bwd`.

float32 or bfloat16 throughout; sums, the saved projections and the bias gradients' sums are float32.  There is no CPU
fallback in `gated_linear`; `GatedLinear` computes the same expression in PyTorch where its input is on the CPU, as the
other modules of a denoiser do.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _lib

_DTYPES = {torch.float32: _lib.DP_DTYPE_F32, torch.bfloat16: _lib.DP_DTYPE_BF16}
_ACTS = {"none": 0, "silu": 1, "gelu": 2}


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
    if not x.is_cuda:
        raise _lib.DiffputerError("gated_linear needs tensors on a CUDA (ROCm) device; there is no CPU fallback")
    raise ValueError("gated_linear takes dense (strided) tensors")


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: torch.Tensor | None = None,
                 b_up: torch.Tensor | None = None, act: str = "silu") -> torch.Tensor:
    """act(x @ w_gate^T + b_gate) * (x @ w_up^T + b_up) -> [..., N].

    x [..., K]; w_gate, w_up [N, K]; b_gate, b_up [N] or None each; all of one dtype (float32 or bfloat16) on one CUDA (ROCm)
    device.  act: "silu", "gelu" (g Phi(g), not its tanh approximation) or "none".  Row strides are used as they are (a column range
    of a wider table is not copied); other layouts are copied.  Runs on torch's current stream of x's device; first
    derivatives only (autocast does not convert its arguments; GatedLinear does), and by backward passes only (a tensor with a forward-mode tangent is refused); not for tracers
    (torch.jit.trace, make_fx, torch.export), which are refused, while torch.compile breaks its graph here; a backward pass under graph capture is refused while a graph of the same leaves, made on a stream
    outside the capture, is alive.  A row of h depends on its own row of x only."""
    code = _ACTS.get(act)
    h = None if code is None else _lib.torch_side().gated_linear(x, w_gate, w_up, b_gate, b_up, code)
    if h is None:
        _refuse(x, w_gate, w_up, b_gate, b_up, act)
    return h


class GatedLinear(nn.Module):
    """`act(gate(x)) * up(x)` with `gate`, `up` two Linear layers in_features -> out_features: a gated layer for denoisers that
    `model.Precond` / `model.Model` take as `denoise_fn`.  State-dict keys `gate.weight`, `gate.bias`, `up.weight`, `up.bias`.

    Under autocast it converts as nn.Linear does: to bf16, or to float32 where autocast asks for float16 (the kernels have no
    float16).  Without autocast x has to be of the parameters' type: `model.Precond` gives its denoiser float32, so a bf16 layer inside
    it needs a denoiser that casts, or autocast."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, act: str = "silu"):
        super().__init__()
        if act not in _ACTS:
            raise ValueError(f"act must be one of {sorted(_ACTS)}, got {act!r}")
        self.gate = nn.Linear(in_features, out_features, bias=bias)
        self.up = nn.Linear(in_features, out_features, bias=bias)
        self.act = act

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.is_cuda:
            args = [x, self.gate.weight, self.up.weight, self.gate.bias, self.up.bias]
            if torch.is_autocast_enabled("cuda"):
                to = torch.bfloat16 if torch.get_autocast_dtype("cuda") == torch.bfloat16 else torch.float32
                args = [t if t is None or t.dtype == torch.float64 else t.to(to) for t in args]
            return gated_linear(*args, act=self.act)
        g = self.gate(x)
        g = nn.functional.silu(g) if self.act == "silu" else nn.functional.gelu(g) if self.act == "gelu" else g
        return g * self.up(x)

    def extra_repr(self) -> str:
        return f"act={self.act}"


__all__ = ["gated_linear", "GatedLinear"]

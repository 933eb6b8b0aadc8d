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


# ---- whether strided tensors share memory, exactly and without the GPU -------------------------------------------------------
# A place of a tensor is base + sum x_k stride_k, 0 <= x_k < n_k, so two tensors meet where a sum of terms with bounded counts takes
# one value.  The largest step first, the counts that are left are those between which the smaller steps can make up the rest: one
# or two at each step where dimensions nest, as a view's do.
_MOST_TRIES = 20_000


def _solutions(terms, total, need):
    """How many ways, up to `need`, there are to write `total` as sum x_k step_k with 0 <= x_k <= most_k; `need` where that takes
    too long to find out.  terms: [(step >= 1, most >= 1)]."""
    terms = sorted(terms, reverse=True)
    reach, common = [0], [0]                                     # of the terms from k on: largest sum, common divisor
    for step, most in reversed(terms):
        reach.append(reach[-1] + step * most)
        common.append(math.gcd(common[-1], step))
    reach, common = reach[::-1], common[::-1]
    tries = 0

    def count(k, left, need):
        nonlocal tries
        tries += 1
        if tries > _MOST_TRIES:
            return need
        if k == len(terms):
            return int(left == 0)
        if left < 0 or left > reach[k] or left % common[k]:
            return 0
        step, most = terms[k]
        found = 0
        for x in range(max(0, -((reach[k + 1] - left) // step)), min(most, left // step) + 1):
            found += count(k + 1, left - x * step, need - found)
            if found >= need:
                return need
        return found

    return count(0, total, need)


def _dims(t):
    return [(s * t.element_size(), n - 1) for s, n in zip(t.stride(), t.shape) if n > 1]


def _meets_itself(t):
    """Whether two elements of t have one place."""
    dims = _dims(t) if t.numel() else []
    if any(s == 0 for s, _ in dims):
        return True
    # differences of two indexes, moved up by n - 1: equal indexes are one solution
    return _solutions([(s, 2 * n) for s, n in dims], sum(s * n for s, n in dims), 2) > 1


def _meet(a, b):
    """Whether a and b, neither of them empty, share a byte."""
    ends = [[(1, t.element_size() - 1)] if t.element_size() > 1 else [] for t in (a, b)]
    back = _dims(b) + ends[1]                                    # counted from b's end
    total = b.data_ptr() - a.data_ptr() + sum(s * n for s, n in back)
    terms = {}
    for s, n in [*_dims(a), *ends[0], *back]:
        if s:
            terms[s] = terms.get(s, 0) + n
    return _solutions(list(terms.items()), total, 1) > 0


def _apart(ts):
    """Whether one look shows that no two of `ts` meet: views with one largest stride, such as column ranges of one table, whose
    places modulo that stride are ranges that do not meet.  (Pair by pair, 100 such views take 50 ms.)"""
    pitches = {max((s for s, _ in _dims(t)), default=0) for t in ts}
    pitch = pitches.pop()
    if pitches or not pitch:
        return False
    last, base = 0, min(t.data_ptr() for t in ts)
    for first, t in sorted((((t.data_ptr() - base) % pitch, t) for t in ts), key=lambda e: e[0]):
        if first < last:
            return False
        last = first + sum(s * n for s, n in _dims(t) if s != pitch) + t.element_size()
    return last <= pitch


def _refuse_shared(grads, what):
    """The error of tensors that cannot be scaled in place, each element once."""
    for i, t in enumerate(grads):
        if any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)) and t.numel():
            raise ValueError(f"{what}: tensor {i} is expanded: its elements share memory")
        if not t.is_contiguous() and _meets_itself(t):
            raise ValueError(f"{what}: tensor {i} overlaps itself: its elements share memory")
    spans = sorted(((t.data_ptr(), t.data_ptr() + sum(s * n for s, n in _dims(t)) + t.element_size(), t) for t in grads if t.numel()), key=lambda e: e[:2])
    groups, reach = [], 0                                        # spans that hang together
    for e in spans:
        if e[0] >= reach:
            groups.append([])
        groups[-1].append(e)
        reach = max(reach, e[1])
    for group in groups:
        if len(group) == 1 or _apart([t for _, _, t in group]):
            continue
        before = []                                              # those that reach behind the start of the next one
        for start, end, t in group:
            before = [e for e in before if e[0] > start]
            if any(_meet(o, t) for _, o in before):
                raise _lib.DiffputerError(f"{what}: two of the tensors share memory")
            before.append((end, t))


def _call(grads, kind, limit, what):
    """The norm; `grads` are clipped in place if there is a limit."""
    call = _lib.torch_side().grads
    norm = call(grads, kind, limit)
    if norm is None:
        _refuse(grads, what)
    if isinstance(norm, int):                                    # tensor number `norm` does not fill one range of memory: copies
        if limit is not None:
            _refuse_shared(grads, what)                          # (of dense tensors only, the library sees it)
        with torch.no_grad():
            flat = [g if i < norm or g.is_contiguous() else g.contiguous() for i, g in enumerate(grads)]
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

    float32 and bfloat16 mix freely; every tensor has to own its elements once (an expanded tensor, one that overlaps itself, or
    two that share memory, are refused; views that interleave without a common element are not).  error_if_nonfinite: wait for the norm, and raise RuntimeError before anything is scaled if it is
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

"""The gated projection (`diffputer_amd.gated`, dp_gated_linear / dp_gated_linear_bwd) on the GPU against its formulas in float64.

Tolerances are componentwise bounds, worked out from the inputs:  a float32 sum of k products is off by at most
gamma(k) = 2 (k + 4) 2^-24 times the sum of the absolute products (2: the matrix pipes may round inside a step of their
own), an elementary function or a rounding in float32 by 2^-22 of its value, and a rounding to the tensor's type by
eps / 2 of it (bf16 2^-8); bf16 keeps the projections for the backward pass in 20 bits (2^-12).  |silu'| <= 1.1, |gelu'| <= 1.13, |silu''| <= 0.5, |gelu''| <= 0.8.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float64
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
E32 = 2.0 ** -22
TINY = 1e-30
A1, A2 = 1.13, 0.8


def gamma(k):
    return 2 * (k + 4) * 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def act_of(g, act):
    """act(g), act'(g) in float64"""
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "gelu":
        p = 0.5 * torch.erfc(-g / math.sqrt(2))
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    return g, torch.ones_like(g)


def make(M, K, N, dtype, bias=True, seed=0, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    x = (torch.randn(M, K, generator=gen) * scale).to(dt)
    w = [(torch.randn(N, K, generator=gen) / math.sqrt(K)).to(dt) for _ in range(2)]
    b = [torch.randn(N, generator=gen).to(dt) if bias else None for _ in range(2)]
    dh = torch.randn(M, N, generator=gen).to(dt)
    return x, w[0], w[1], b[0], b[1], dh


class Ref:
    """Formulas and error bounds in float64 on the CPU."""

    def __init__(self, x, wg, wu, bg, bu, dh, act):
        dt = x.dtype
        u_t = half_step(dt)
        mix = u_t if dt == torch.bfloat16 else 0.0                # dg, du are rounded to bf16 as operands
        kept = 2.0 ** -12 if dt == torch.bfloat16 else 0.0        # the saved projections
        x, wg, wu, dh = (t.detach().cpu().to(F8) for t in (x, wg, wu, dh))
        N, K = wg.shape
        M = x.shape[0]
        zero = torch.zeros(N, dtype=F8)
        bg, bu = (zero if b is None else b.detach().cpu().to(F8) for b in (bg, bu))
        g, u = x @ wg.T + bg, x @ wu.T + bu
        eg, eu = (gamma(K) * (x.abs() @ w.abs().T + b.abs()) for w, b in ((wg, bg), (wu, bu)))
        a, da = act_of(g, act)
        ea = A1 * eg + E32 * a.abs()
        self.h = a * u
        self.eh = ea * (u.abs() + eu) + a.abs() * eu + (E32 + u_t) * self.h.abs() * 1.01 + TINY
        du, dg = dh * a, dh * u * da
        eg, eu = eg + kept * (g.abs() + eg), eu + kept * (u.abs() + eu)
        ea = A1 * eg + E32 * a.abs()
        edu = dh.abs() * ea + E32 * du.abs()
        edg = dh.abs() * (eu * A1 + (u.abs() + eu) * (A2 * eg + 2 * E32 * A1)) + 2 * E32 * dg.abs()
        rdu, rdg = edu + mix * (du.abs() + edu), edg + mix * (dg.abs() + edg)      # as operands of the products
        self.dx = dg @ wg + du @ wu
        mag = (dg.abs() + rdg) @ wg.abs() + (du.abs() + rdu) @ wu.abs()
        self.edx = rdg @ wg.abs() + rdu @ wu.abs() + gamma(2 * N) * mag + u_t * (self.dx.abs() + rdg @ wg.abs() + rdu @ wu.abs()) + TINY
        for name, d, r, e in (("g", dg, rdg, edg), ("u", du, rdu, edu)):
            v = d.T @ x
            err = r.T @ x.abs() + gamma(M) * ((d.abs() + r).T @ x.abs())
            setattr(self, "dw" + name, v)
            setattr(self, "edw" + name, err + u_t * (v.abs() + err) + TINY)
            s = d.sum(0)
            err = e.sum(0) + gamma(M) * (d.abs() + e).sum(0)
            setattr(self, "db" + name, s)
            setattr(self, "edb" + name, err + u_t * (s.abs() + err) + TINY)


def close(got, want, bound, what):
    assert tuple(got.shape) == tuple(want.shape), (what, got.shape, want.shape)
    off = (got.detach().cpu().to(F8) - want).abs()
    assert torch.isfinite(got.detach().cpu().to(F8)).all(), what
    worst = float((off / bound).max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"


def check(x, wg, wu, bg, bu, dh, act, train=True):
    from diffputer_amd.gated import gated_linear
    ref = Ref(x, wg, wu, bg, bu, dh, act)
    dev = [None if t is None else t.to(DEV) for t in (x, wg, wu, bg, bu)]
    close(gated_linear(*dev, act=act), ref.h, ref.eh, "h")
    if not train:
        return
    leaves = [None if t is None else t.requires_grad_() for t in dev]
    h = gated_linear(*leaves, act=act)
    close(h, ref.h, ref.eh, "h (training)")
    given = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(h, given, dh.to(DEV)))
    for name in ("x", "wg", "wu", "bg", "bu"):
        if {"bg": bg, "bu": bu}.get(name, x) is not None:
            g = next(grads)
            assert g.dtype == x.dtype
            close(g, getattr(ref, "d" + name), getattr(ref, "ed" + name), "d" + name)


SIZES = [  # M, K, N
    (1, 1, 1), (1, 64, 64), (1, 256, 520), (2, 7, 3), (3, 8, 16), (15, 9, 64), (16, 64, 32), (17, 65, 33), (31, 130, 31),
    (33, 72, 100), (64, 128, 128), (1, 1000, 4100), (20, 520, 4100), (50, 1032, 300), (64, 2050, 4096), (65, 63, 129), (100, 200, 65), (130, 320, 260), (257, 100, 40), (300, 33, 257), (1000, 16, 8),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_against_formula(M, K, N, dtype):
    check(*make(M, K, N, dtype, seed=M * 7 + K + N), act="silu")


@pytest.fixture
def tune():
    from diffputer_amd import _lib
    lib = _lib.load()

    def put(kernel, splits):
        _lib.check(lib.dp_tune(b"gated_kernel", kernel), "dp_tune")
        _lib.check(lib.dp_tune(b"gated_splits", splits), "dp_tune")

    yield put
    put(0, 0)


@pytest.mark.parametrize("M,K,N", [(1, 8, 8), (40, 64, 64), (70, 200, 40), (129, 64, 65), (257, 72, 129), (300, 136, 264), (513, 1032, 264), (600, 71, 300)])
@pytest.mark.parametrize("kernel,splits", [(1, 0), (1, 3), (128, 0), (128, 1), (128, 3), (256, 0), (256, 1), (256, 5)])
def test_every_kernel(tune, kernel, splits, M, K, N):
    tune(kernel, splits)
    check(*make(M, K, N, "bf16", seed=M + K), act="silu")


@pytest.mark.parametrize("M,K,N", [(1, 8, 8), (40, 64, 64), (70, 200, 40), (129, 64, 65), (257, 73, 129), (300, 136, 264), (513, 1032, 264), (200, 31, 66)])
@pytest.mark.parametrize("kernel,splits", [(1, 0), (1, 3), (64, 0), (64, 1), (64, 4), (128, 0), (128, 1), (128, 3)])
def test_every_kernel_f32(tune, kernel, splits, M, K, N):
    tune(kernel, splits)
    check(*make(M, K, N, "f32", seed=M + K), act="silu")


@pytest.mark.parametrize("kernel,dtype", [(1, "bf16"), (128, "bf16"), (256, "bf16"), (1, "f32"), (64, "f32"), (128, "f32")])
def test_every_kernel_strides(tune, kernel, dtype):
    """A column range of a wider table (the columns beside it hold NaN): aligned rows are read where they are, others copied or
    read by narrower loads."""
    from diffputer_amd.gated import gated_linear
    tune(kernel, 0)
    x, wg, wu, bg, bu, dh = make(300, 72, 136, dtype, seed=6)
    ref = Ref(x, wg, wu, bg, bu, dh, "silu")
    for off in (0, 8, 3):
        wide = torch.full((300, 96), float("nan"), dtype=x.dtype, device=DEV)
        wide[:, off:off + 72] = x.to(DEV)
        leaves = [wide[:, off:off + 72], *[t.to(DEV) for t in (wg, wu, bg, bu)]]
        leaves = [t.detach().requires_grad_() for t in leaves]
        h = gated_linear(*leaves)
        close(h, ref.h, ref.eh, "h")
        for name, g in zip(("x", "wg", "wu", "bg", "bu"), torch.autograd.grad(h, leaves, dh.to(DEV))):
            close(g, getattr(ref, "d" + name), getattr(ref, "ed" + name), "d" + name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kernel", [0, 1, 128])
def test_some_gradients_on_every_kernel(tune, kernel, dtype):
    """dx alone, one weight's gradient alone, both: the products run in other launches than all together."""
    from diffputer_amd.gated import gated_linear
    tune(kernel, 0)
    x, wg, wu, bg, bu, dh = make(300, 72, 136, dtype, seed=7)
    ref = Ref(x, wg, wu, bg, bu, dh, "silu")
    names = ("x", "wg", "wu", "bg", "bu")
    for want in ((0,), (1,), (2,), (1, 2), (0, 2), (3,), (0, 1, 2)):
        dev = [t.to(DEV) for t in (x, wg, wu, bg, bu)]
        for i in want:
            dev[i].requires_grad_()
        for i, g in zip(want, torch.autograd.grad(gated_linear(*dev), [dev[i] for i in want], dh.to(DEV))):
            close(g, getattr(ref, "d" + names[i]), getattr(ref, "ed" + names[i]), "d" + names[i])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
@pytest.mark.parametrize("bias", [True, False])
def test_activations_and_bias(act, bias, dtype):
    check(*make(70, 96, 72, dtype, bias=bias, seed=3, scale=3.0), act=act)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(512, 1024, 768), (1024, 512, 1000), (2048, 264, 256), (700, 1030, 520)])
def test_larger(M, K, N, dtype):
    check(*make(M, K, N, dtype, seed=5), act="silu")


def test_one_bias_only():
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, dh = make(20, 40, 24, "f32", seed=8)
    for b0, b1 in ((bg, None), (None, bu)):
        ref = Ref(x, wg, wu, b0, b1, dh, "silu")
        dev = [None if t is None else t.to(DEV).requires_grad_() for t in (x, wg, wu, b0, b1)]
        h = gated_linear(*dev)
        close(h, ref.h, ref.eh, "h")
        given = [t for t in dev if t is not None]
        db = torch.autograd.grad(h, given, dh.to(DEV))[-1]
        name = "bg" if b1 is None else "bu"
        close(db, getattr(ref, "d" + name), getattr(ref, "ed" + name), name)


@pytest.mark.parametrize("act,at", [("silu", -200.0), ("silu", 200.0), ("silu", -20.0), ("gelu", -200.0), ("gelu", 200.0), ("gelu", -6.0), ("gelu", -13.0)])
def test_saturated_gates(act, at):
    """Gates far out: the exponentials overflow or vanish, values and gradients stay what the formula says."""
    x, wg, wu, bg, bu, dh = make(40, 16, 24, "f32", seed=9)
    bg = torch.full_like(bg, at)
    check(x, wg, wu, bg, bu, dh, act)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_differences(dtype):
    """The gradients against central differences of the formula in float64 along a random direction."""
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, dh = make(33, 24, 20, dtype, seed=11)
    ref = Ref(x, wg, wu, bg, bu, dh, "gelu")
    leaves = [t.to(DEV).requires_grad_() for t in (x, wg, wu, bg, bu)]
    grads = torch.autograd.grad(gated_linear(*leaves, act="gelu"), leaves, dh.to(DEV))
    gen = torch.Generator().manual_seed(1)
    at = [t.to(F8) for t in (x, wg, wu, bg, bu)]
    v = [torch.randn(t.shape, generator=gen, dtype=F8) for t in at]

    def loss(eps):
        p = [t + eps * d for t, d in zip(at, v)]
        return float((act_of(p[0] @ p[1].T + p[3], "gelu")[0] * (p[0] @ p[2].T + p[4]) * dh.to(F8)).sum())

    eps = 1e-4
    slope = (loss(eps) - loss(-eps)) / (2 * eps)
    half = (loss(2 * eps) - loss(-2 * eps)) / (4 * eps)
    truncation = abs(half - slope)                                  # about 3 times the error of `slope` in eps^2
    ours = sum(float((g.cpu().to(F8) * d).sum()) for g, d in zip(grads, v))
    bound = sum(float((getattr(ref, "ed" + n) * d.abs()).sum()) for n, d in zip(("x", "wg", "wu", "bg", "bu"), v))
    assert abs(ours - slope) <= bound + truncation + 1e-6 * abs(slope), (ours, slope, bound, truncation)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_layouts(dtype):
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, dh = make(50, 72, 40, dtype, seed=13)
    want = gated_linear(*[t.to(DEV) for t in (x, wg, wu, bg, bu)])
    wide = torch.full((50, 100), float("nan"), dtype=x.dtype, device=DEV)
    for off in (0, 3, 8, 28):                                       # a column range of a wider table
        wide[:] = float("nan")
        wide[:, off:off + 72] = x.to(DEV)
        assert torch.equal(gated_linear(wide[:, off:off + 72], *[t.to(DEV) for t in (wg, wu, bg, bu)]), want), off
    fused = torch.cat([wg, wu]).to(DEV)                             # both weights as halves of one tensor
    assert torch.equal(gated_linear(x.to(DEV), fused[:40], fused[40:], bg.to(DEV), bu.to(DEV)), want)
    pair = torch.stack([wg, wu], 1).to(DEV)                         # rows of both in turn: row stride 2 K
    assert torch.equal(gated_linear(x.to(DEV), pair[:, 0], pair[:, 1], bg.to(DEV), bu.to(DEV)), want)
    assert torch.equal(gated_linear(x.to(DEV), pair[:, 0], wu.to(DEV), bg.to(DEV), bu.to(DEV)), want)      # two row strides
    assert torch.equal(gated_linear(x.t().contiguous().to(DEV).t(), *[t.to(DEV) for t in (wg, wu, bg, bu)]), want)
    assert torch.equal(gated_linear(x.to(DEV).reshape(5, 2, 5, 72), *[t.to(DEV) for t in (wg, wu, bg, bu)]), want.reshape(5, 2, 5, 40))
    one = gated_linear(x[0].to(DEV), *[t.to(DEV) for t in (wg, wu, bg, bu)])
    assert one.shape == (40,)
    row = gated_linear(x[:1].to(DEV).expand(50, 72), *[t.to(DEV) for t in (wg, wu, bg, bu)])               # one row, broadcast
    assert torch.equal(row, row[:1].expand_as(row))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gradients_of_broadcast_and_shared_inputs(dtype):
    """An expanded x, one weight used as gate and as up weight, and an expanded dh (h.sum().backward())."""
    from diffputer_amd.gated import gated_linear
    x, w, _, b, _, _ = make(1, 24, 16, dtype, seed=14)
    n = 5
    xs = x.expand(n, 24)
    ones = torch.ones(n, 16, dtype=x.dtype)
    ref = Ref(xs, w, w, b, b, ones, "silu")
    lx, lw, lb = (t.to(DEV).requires_grad_() for t in (x, w, b))
    gated_linear(lx.expand(n, 24), lw, lw, lb, lb).sum().backward()
    u = half_step(x.dtype)
    for got, v, e in ((lx.grad, ref.dx.sum(0, keepdim=True), ref.edx.sum(0, keepdim=True)), (lw.grad, ref.dwg + ref.dwu, ref.edwg + ref.edwu),
                      (lb.grad, ref.dbg + ref.dbu, ref.edbg + ref.edbu)):
        close(got, v, e + 2 * n * u * (ref_abs(v) + e), "shared")   # torch adds the parts in the tensor's type


def ref_abs(v):
    return v.abs() + float(v.abs().max())


def test_only_the_wanted_gradients():
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, dh = make(30, 20, 12, "f32", seed=15)
    ref = Ref(x, wg, wu, bg, bu, dh, "silu")
    for i, name in enumerate(("x", "wg", "wu", "bg", "bu")):
        dev = [t.to(DEV) for t in (x, wg, wu, bg, bu)]
        dev[i].requires_grad_()
        (g,) = torch.autograd.grad(gated_linear(*dev), [dev[i]], dh.to(DEV))
        close(g, getattr(ref, "d" + name), getattr(ref, "ed" + name), name)


def test_first_derivatives_only():
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, dh = make(20, 12, 8, "f32", seed=16)
    leaves = [t.to(DEV).requires_grad_() for t in (x, wg, wu, bg, bu)]
    plain = torch.autograd.grad(gated_linear(*leaves), leaves, dh.to(DEV))
    grads = torch.autograd.grad(gated_linear(*leaves), leaves, dh.to(DEV), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, grads))
    with pytest.raises(RuntimeError):                               # the second graph does not lead to a leaf
        torch.autograd.grad(grads[0].sum(), leaves[1], retain_graph=True)
    with pytest.raises(RuntimeError, match="first derivatives only"):
        grads[0].sum().backward()


def test_changed_inputs_are_noticed():
    """autograd refuses a backward pass whose saved inputs were overwritten in between."""
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, dh = [t.to(DEV) for t in make(20, 12, 8, "f32", seed=16)]
    wg.requires_grad_()
    h = gated_linear(x, wg, wu, bg, bu)
    x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h, wg, dh)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_no_rows(dtype):
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, _ = make(3, 24, 16, dtype)
    leaves = [t.to(DEV).requires_grad_() for t in (x[:0], wg, wu, bg, bu)]
    h = gated_linear(*leaves)
    assert h.shape == (0, 16)
    grads = torch.autograd.grad(h, leaves, torch.empty_like(h))
    assert grads[0].shape == (0, 24)
    assert all(bool((g == 0).all()) for g in grads[1:])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(40, 72, 33), (1, 64, 64), (300, 128, 256)])
def test_nan_and_inf_stay_in_their_rows(M, K, N, dtype):
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, _ = [t.to(DEV) for t in make(M, K, N, dtype, seed=17)]
    want = gated_linear(x, wg, wu, bg, bu)
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[M // 2, K - 1] = bad
        h = gated_linear(y, wg, wu, bg, bu)
        keep = torch.arange(M, device=DEV) != M // 2
        assert torch.equal(h[keep], want[keep])
        assert not torch.isfinite(h[M // 2]).any()
    v = wg.clone()
    v[N - 1, 0] = float("nan")                                      # a weight row: its column of h
    h = gated_linear(x, v, wu, bg, bu)
    assert torch.isnan(h[:, N - 1]).all() and torch.equal(h[:, :N - 1], want[:, :N - 1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,N", [(1, 24), (37, 33), (130, 64), (300, 264)])
def test_nothing_beside_the_output_is_written(M, N, dtype):
    """h as a block of a larger buffer through the C ABI: the rows behind the last one and the columns beside it stay."""
    import ctypes as C

    from diffputer_amd import _lib
    from diffputer_amd.gated import _DTYPES, gated_linear
    K = 40
    x, wg, wu, bg, bu, _ = [t.to(DEV) for t in make(M, K, N, dtype, seed=19)]
    want = gated_linear(x, wg, wu, bg, bu)
    lib = _lib.load()
    buf = torch.full((M + 9, N + 13), 7.0, dtype=x.dtype, device=DEV)
    ops = (_DTYPES[x.dtype], x.data_ptr(), K, wg.data_ptr(), wu.data_ptr(), K)
    need = lib.dp_gated_linear_workspace_bytes(*ops, M, N, K, 0)
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    h = buf[3:3 + M, 5:5 + N]
    rc = lib.dp_gated_linear(*ops, bg.data_ptr(), bu.data_ptr(), h.data_ptr(), N + 13, None,
                             M, N, K, 1, ws.data_ptr(), need, C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0, lib.dp_last_error()
    assert torch.equal(h, want)
    h.fill_(7.0)
    assert bool((buf == 7.0).all())


def test_offsets_past_32_bits():
    """More than 2^31 elements of h: the last rows against the formula, and weight gradients that only they contribute to."""
    from diffputer_amd.gated import gated_linear
    M, K, N, tail = 270_000, 64, 8192, 70
    x, wg, wu, bg, bu, dh = make(tail, K, N, "bf16", seed=23)
    ref = Ref(x, wg, wu, bg, bu, dh, "silu")
    big = torch.full((M, K), 0.5, dtype=torch.bfloat16, device=DEV)
    big[-tail:] = x.to(DEV)
    leaves = [big.requires_grad_(), *[t.to(DEV).requires_grad_() for t in (wg, wu, bg, bu)]]
    h = gated_linear(*leaves)
    close(h[-tail:], ref.h, ref.eh, "h")
    d = torch.zeros((M, N), dtype=torch.bfloat16, device=DEV)
    d[-tail:] = dh.to(DEV)
    grads = torch.autograd.grad(h, leaves, d)
    close(grads[0][-tail:], ref.dx, ref.edx, "dx")
    assert not grads[0][:-tail].any()
    for name, g in zip(("wg", "wu", "bg", "bu"), grads[1:]):
        # sums of M terms, all but `tail` of them zero: the bound counts additions, of zeros too
        more = gamma(M) / gamma(tail)
        close(g, getattr(ref, "d" + name), more * getattr(ref, "ed" + name), "d" + name)
    del h, d, grads, big, leaves
    torch.cuda.empty_cache()


@torch.no_grad()
def test_general_kernel_more_than_2_20_tiles(tune):
    """A grid that is folded: equal rows give equal results everywhere, the last rows their own."""
    from diffputer_amd.gated import gated_linear
    M, K, N, tail = 270_000, 64, 8192, 70
    x, wg, wu, bg, bu, dh = make(tail, K, N, "bf16", seed=29)
    ref = Ref(x, wg, wu, bg, bu, dh, "silu")
    big = torch.full((M, K), 0.5, dtype=torch.bfloat16, device=DEV)
    big[-tail:] = x.to(DEV)
    tune(1, 0)
    h = gated_linear(big, *[t.to(DEV) for t in (wg, wu, bg, bu)])
    close(h[-tail:], ref.h, ref.eh, "h")
    for a in range(0, M - tail, 30_000):
        assert torch.equal(h[a:min(a + 30_000, M - tail)], h[:1].expand(min(30_000, M - tail - a), N))
    del h, big
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_two_threads(dtype):
    """Two threads, each with a stream of its own, at the same time."""
    import threading

    from diffputer_amd.gated import gated_linear
    sets = [[t.to(DEV) for t in make(200 + 100 * i, 136, 96, dtype, seed=40 + i)] for i in range(2)]
    want = [gated_linear(*s[:5]) for s in sets]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    leaves = [t.detach().requires_grad_() for t in sets[i][:5]]
                    h = gated_linear(*leaves)
                    torch.autograd.grad(h, leaves, sets[i][5])
                got[i] = h.detach()
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_same_bits_twice(dtype):
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, dh = [t.to(DEV) for t in make(900, 200, 136, dtype, seed=21)]
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]

    def once():
        h = gated_linear(*leaves)
        return [h.detach(), *torch.autograd.grad(h, leaves, dh)]

    first = once()
    for _ in range(3):
        torch.randn(1 << 20, device=DEV)
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


def test_side_stream():
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, dh = [t.to(DEV) for t in make(600, 256, 200, "bf16", seed=22)]
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    h = gated_linear(*leaves)
    want = [h.detach(), *torch.autograd.grad(h, leaves, dh)]
    del h                                                           # its graph: a leaf's accumulation node belongs to one stream
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        h = gated_linear(*leaves)
        got = [h.detach(), *torch.autograd.grad(h, leaves, dh)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype,M", [("bf16", 1), ("bf16", 300), ("f32", 70)])
def test_captured_and_replayed(dtype, M):
    """Forward and backward in a graph, replayed with new inputs and eager work between the replays; a second graph of the
    same operator beside it."""
    from diffputer_amd.gated import gated_linear
    K, N = 96, 72
    sets = [make(M, K, N, dtype, seed=30 + i) for i in range(3)]
    static = [t.to(DEV) for t in sets[0]]
    leaves = [t.requires_grad_() for t in static[:5]]

    def once():
        h = gated_linear(*leaves)
        return [h.detach(), *torch.autograd.grad(h, leaves, static[5])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        once()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = once()
        graphs.append((g, out))
    for it in range(6):
        with torch.no_grad():
            for t, v in zip(static, sets[it % 3]):
                t.copy_(v.to(DEV))
        want = once()
        torch.cuda.synchronize()
        for g, out in graphs:
            g.replay()
            once()                                                  # eager work of its own in between
        torch.cuda.synchronize()
        for g, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(want, out)), it


@pytest.mark.parametrize("N,K", [((1 << 20) + 1, 1), ((1 << 32) + 5, 1), (1, (1 << 20) + 8), (3, (1 << 32) + 7)])
def test_too_wide_is_refused(N, K):
    """Sizes that the C ABI does not take, beyond 32 bits among them (nothing is allocated: expanded tensors)."""
    from diffputer_amd._lib import DiffputerError
    from diffputer_amd.gated import gated_linear
    one = torch.ones(1, 1, dtype=torch.bfloat16, device=DEV)
    for grad in (False, True):
        with pytest.raises(DiffputerError, match="2\\^20"):
            gated_linear(one.expand(2, K).detach().requires_grad_(grad), one.expand(N, K), one.expand(N, K))


def test_graphs_of_two_streams_are_seen():
    """A leaf's accumulation node stays with the stream of its first graph as long as a graph of the leaf lives."""
    from diffputer_amd import _lib
    from diffputer_amd.gated import gated_linear
    elsewhere = _lib.torch_side().goes_elsewhere
    x, wg, wu, bg, bu, dh = [t.to(DEV) for t in make(70, 96, 72, "bf16", seed=51)]
    leaves = [t.requires_grad_() for t in (wg, wu, bg, bu)]
    h = gated_linear(x, *leaves)
    assert elsewhere(h) is False
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        k = gated_linear(x, *leaves)
        assert elsewhere(k) is True
        del k
        other = gated_linear(x.detach().requires_grad_(), *[t.detach().requires_grad_() for t in leaves])
        assert elsewhere(other) is False
    torch.cuda.current_stream().wait_stream(s)
    del h
    with torch.cuda.stream(s):
        k = gated_linear(x, *leaves)
        assert elsewhere(k) is False
    torch.cuda.synchronize()


def test_capture_beside_an_eager_graph_is_refused():
    """A backward pass is not captured while an eager graph of the same leaves lives; the process goes on, and without that
    graph the capture works, with .backward() too."""
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, dh = [t.to(DEV) for t in make(70, 96, 72, "bf16", seed=52)]
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    eager = gated_linear(*leaves)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="drop that graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(gated_linear(*leaves), leaves, dh)
    want = [g.clone() for g in torch.autograd.grad(eager, leaves, dh)]
    del eager
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        gated_linear(*leaves).backward(dh)
    torch.cuda.current_stream().wait_stream(s)
    for t in leaves:
        t.grad.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gated_linear(*leaves).backward(dh)
    for _ in range(3):
        for t in leaves:
            t.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))


def test_module_and_denoiser_training_step():
    """A denoiser of gated layers inside model.Model: loss, gradients, clipping and Adam's step on the GPU against the same
    modules on the CPU in float64 (the draws replayed)."""
    from diffputer_amd.gated import GatedLinear
    from diffputer_amd.grads import clip_grads
    from diffputer_amd.model import Model, PositionalEmbedding

    class Denoiser(torch.nn.Module):
        def __init__(self, d, h):
            super().__init__()
            self.proj = GatedLinear(d, h)
            self.map_noise = PositionalEmbedding(num_channels=h)
            self.mid = GatedLinear(h, 2 * h, act="gelu")
            self.out = torch.nn.Linear(2 * h, d)

        def forward(self, x, noise_labels, class_labels=None):
            return self.out(self.mid(self.proj(x) + self.map_noise(noise_labels).to(x.dtype)))

    d, h, n = 9, 64, 200
    torch.manual_seed(5)
    cpu = Model(denoise_fn=Denoiser(d, h), hid_dim=d)
    gpu = Model(denoise_fn=Denoiser(d, h), hid_dim=d)
    gpu.load_state_dict(cpu.state_dict())
    assert "denoise_fn_D.denoise_fn_F.mid.gate.weight" in gpu.state_dict()
    gpu = gpu.to(DEV)
    x, zs, zn = torch.randn(n, d), torch.randn(n), torch.randn(n, d)

    def step(model, dev, limit):
        saved = (torch.randn, torch.randn_like)
        torch.randn = lambda *a, **k: zs.to(dev)
        torch.randn_like = lambda t, **k: zn.to(dev)
        try:
            loss = model(x.to(dev))
        finally:
            torch.randn, torch.randn_like = saved
        params = list(model.parameters())
        for p in params:
            p.grad = None
        loss.backward()
        before = [p.grad.clone() for p in params]
        norm = clip_grads([p.grad for p in params], limit) if dev != "cpu" else torch.nn.utils.clip_grad_norm_(params, limit)
        after = [p.grad.clone() for p in params]
        torch.optim.Adam(params, lr=1e-3).step()
        return float(loss.detach()), before, float(norm), after

    ref = step(cpu, "cpu", 0.25)
    got = step(gpu, DEV, 0.25)
    assert abs(got[0] - ref[0]) <= 1e-4 * abs(ref[0])
    assert ref[2] > 0.25, "the limit has to bite"
    # both sides are float32 with sums of a few hundred terms in different orders: 1e-4 of a tensor's scale is over 1000 half steps
    for i in (1, 3):
        for a, b in zip(got[i], ref[i]):
            assert float((a.cpu() - b).abs().max()) <= 1e-4 * float(b.abs().max()) + 1e-8
    assert abs(got[2] - ref[2]) <= 1e-4 * ref[2]
    total = math.sqrt(sum(float(g.double().square().sum()) for g in got[3]))
    assert abs(total - 0.25) <= 1e-5


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("kernel", [0, 128, 256])
def test_every_bf16_gate(kernel, act, tune):
    """act and act' at every finite bf16 number of at most 100: x = g, Wg = 1, u = bu = 1, dh = 1, so that h = act(g),
    dbu's terms are act(g) and dx = act'(g).

    Beside the bounds above: the hardware's 2^x and reciprocal (2^-17 of sigmoid), Phi's fit and exponential (2^-16 of it); gates are
    kept in 20 bits exactly.  dx is rounded twice, as the product's operand and as the output.  Behind |g| = 13 gelu's left tail is below 1e-37, and
    results below float32's smallest normal number, 1.2e-38, may be 0."""
    from diffputer_amd.gated import gated_linear
    tune(kernel, 0)
    g = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    g = g[g.abs() <= 100].reshape(-1, 1)
    one, zero = torch.ones(1, 1, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.bfloat16)
    leaves = [t.to(DEV).requires_grad_() for t in (g, one, zero, zero[0], one[0])]
    h = gated_linear(*leaves, act=act)
    dx = torch.autograd.grad(h, leaves, torch.ones_like(h))[0]
    a, da = act_of(g.to(F8), act)
    e, tail = 2.0 ** -16, 2e-37 * (1 + g.to(F8).abs())
    step = half_step(torch.bfloat16)
    close(h, a, (e + step) * 1.01 * a.abs() + tail, "h")
    eda = e * (1 + g.to(F8).abs() * (1 - torch.sigmoid(g.to(F8)).clamp(max=1))) * torch.sigmoid(g.to(F8)) if act == "silu" else e * (0.5 * torch.erfc(-g.to(F8) / math.sqrt(2)) + g.to(F8).abs() * torch.exp(-g.to(F8) ** 2 / 2))
    close(dx, da, (eda + 2 * step * da.abs()) * 1.02 + tail, "dx")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(32, 4096, 8192), (33, 2048, 4104), (40, 1024, 8200), (64, 4096, 2056), (47, 2056, 4097), (64, 1032, 2100), (33, 1027, 2048)])
def test_some_rows_of_large_layers(M, K, N, dtype):
    """Where the kernel for few rows and the tile kernels take turns."""
    check(*make(M, K, N, dtype, seed=M + N), act="silu", train=M != 32)


def test_no_tangent_is_lost():
    """Forward-mode derivatives on the device: refused with and without gradients, through the module too."""
    from torch.autograd import forward_ad

    from diffputer_amd._lib import DiffputerError
    from diffputer_amd.gated import GatedLinear, gated_linear
    from diffputer_amd.grads import clip_grads, grad_norm
    layer = GatedLinear(8, 16).to(DEV)
    x = torch.randn(3, 8, device=DEV)
    want = layer(x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (layer, lambda t: gated_linear(t, layer.gate.weight.detach(), layer.up.weight.detach()), lambda t: grad_norm([t]), lambda t: clip_grads([t], 1e-3)):
            with pytest.raises(DiffputerError, match="forward-mode"):
                call(dual)
        assert torch.equal(layer(x), want)
        with torch.inference_mode():
            assert torch.equal(layer(x), want)
    assert torch.equal(layer(x), want)


def test_traces_on_the_device():
    """Tracers are refused; a mode that only watches, and torch.compile, which breaks its graph, run the kernels."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode

    from diffputer_amd._lib import DiffputerError
    from diffputer_amd.gated import GatedLinear
    layer = GatedLinear(8, 16).to(DEV).requires_grad_(False)
    x = torch.randn(3, 8, device=DEV)
    want = layer(x)
    for trace in (lambda: torch.jit.trace(layer, (x,)), lambda: make_fx(layer)(x)):
        with pytest.raises(DiffputerError, match="traced"):
            trace()
    with FlopCounterMode(display=False):
        assert torch.equal(layer(x), want)
    assert torch.equal(torch.compile(layer, backend="eager")(x), want)
    assert torch.equal(layer(x), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("which", [0, 1, 2, 3, 4, 5])
def test_lazily_negated_tensors(which, dtype):
    """A tensor whose negation is a bit (as the imaginary part of a conjugate has it) is read with its sign, dense or not."""
    from diffputer_amd.gated import gated_linear
    sets = [t.to(DEV) for t in make(9, 16, 8, dtype, seed=60 + which)]

    lazy, plain = list(sets), list(sets)
    lazy[which], plain[which] = torch._neg_view(sets[which]), -sets[which]
    assert lazy[which].is_neg() and not plain[which].is_neg()
    others = [i for i in range(5) if i != which]

    def once(t):
        leaves = [v.detach().requires_grad_(i in others) for i, v in enumerate(t[:5])]
        h = gated_linear(*leaves)
        return [h.detach(), *torch.autograd.grad(h, [leaves[i] for i in others], t[5])]

    assert all(torch.equal(a, b) for a, b in zip(once(lazy), once(plain)))
    with torch.no_grad():
        assert torch.equal(gated_linear(*lazy[:5]), gated_linear(*plain[:5]))


def test_lazily_negated_column():
    """A column of one imaginary part per row: strided, and one element wide."""
    from diffputer_amd.gated import gated_linear
    z = torch.randn(20, 1, dtype=torch.complex64, device=DEV)
    w = torch.randn(8, 1, device=DEV)
    lazy = z.conj().imag
    assert lazy.is_neg()
    assert torch.equal(gated_linear(lazy, w, w), gated_linear(-z.imag.clone(), w, w))


@pytest.mark.parametrize("act", ["silu", "none"])
def test_module_under_autocast(act):
    """GatedLinear converts under autocast as the Linear layers that it has on the CPU do: bf16 there, float32 where autocast asks for
    float16, which the kernels do not have; gradients arrive in the parameters' own type."""
    from diffputer_amd.gated import GatedLinear, gated_linear
    torch.manual_seed(2)
    layer = GatedLinear(24, 40, act=act).to(DEV)
    x = torch.randn(50, 24, device=DEV)
    params = list(layer.parameters())
    plain = layer(x)
    low = [t.detach().bfloat16().requires_grad_() for t in (x, layer.gate.weight, layer.up.weight, layer.gate.bias, layer.up.bias)]
    want = gated_linear(*low, act=act)
    dh = torch.randn(50, 40, device=DEV).bfloat16()
    grads = torch.autograd.grad(want, [low[1], low[3], low[2], low[4], low[0]], dh)
    for given in (x.clone(), x.bfloat16()):
        given.requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            h = layer(given)
        assert h.dtype == torch.bfloat16 and torch.equal(h, want)
        got = torch.autograd.grad(h, [*params, given], dh)
        assert all(g.dtype == p.dtype and torch.equal(g, w.to(p.dtype)) for g, p, w in zip(got, [*params, given], grads))
    with torch.autocast("cuda", dtype=torch.float16):
        assert torch.equal(layer(x), plain) and torch.equal(layer(x.half()), layer(x.half().float()))
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.autocast("cuda", enabled=False):
        assert torch.equal(layer(x), plain)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert torch.equal(layer(x), plain)
    with pytest.raises(ValueError, match="float64"), torch.autocast("cuda", dtype=torch.bfloat16):
        layer(x.double())


def test_captured_backward_over_a_forked_stream():
    """A stream that is forked inside the capture is part of it: gradients may go to a node that was made there."""
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, dh = [t.to(DEV) for t in make(70, 96, 72, "f32", seed=54)]
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    side = torch.cuda.Stream()

    def once():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            w = leaves[1] * 2                                       # its node, and the leaf's, belong to the side stream
        main.wait_stream(side)
        h = gated_linear(leaves[0], w, *leaves[2:])
        return [h.detach(), *torch.autograd.grad(h, leaves, dh)]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        want = [t.clone() for t in once()]
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = once()
    for _ in range(4):
        for t in out:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        torch.randn(1 << 16, device=DEV).sum()


def test_capture_beside_a_graph_of_a_side_stream_is_refused():
    """The same with a living graph of the leaves on a stream that is no part of the capture; the process goes on."""
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, dh = [t.to(DEV) for t in make(70, 96, 72, "bf16", seed=55)]
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        eager = gated_linear(*leaves)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="drop that graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(gated_linear(*leaves), leaves, dh)
    with torch.cuda.stream(s):
        want = torch.autograd.grad(eager, leaves, dh)
    torch.cuda.synchronize()
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = torch.autograd.grad(gated_linear(*leaves), leaves, dh)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_two_threads_every_result(dtype):
    """Two threads on streams of their own: h and every gradient of every call, with sizes that are copied to aligned rows, split into
    slices and joined, and small ones, so that workspaces of both threads are written at the same time."""
    import threading

    from diffputer_amd.gated import gated_linear
    sizes = [[(300, 513, 520), (200, 4096, 96), (40, 72, 33)], [(600, 1032, 264), (310, 511, 500), (129, 64, 65)]]
    sets = [[[t.to(DEV) for t in make(*z, dtype, seed=70 + 10 * i + j)] for j, z in enumerate(s)] for i, s in enumerate(sizes)]

    def once(s):
        leaves = [t.detach().requires_grad_() for t in s[:5]]
        h = gated_linear(*leaves)
        return [h.detach(), *torch.autograd.grad(h, leaves, s[5])]

    want = [[once(s) for s in per] for per in sets]
    torch.cuda.synchronize()
    wrong, errors = [None, None], []
    together = threading.Barrier(2)

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                bad = torch.zeros((), dtype=torch.int64, device=DEV)
                together.wait(60)
                for _ in range(40):
                    for s, w in zip(sets[i], want[i]):
                        for a, b in zip(once(s), w):
                            bad += (a != b).sum()
                wrong[i] = int(bad)
        except Exception as e:                                      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert wrong == [0, 0]


def test_float32_offsets_past_32_bits():
    """More than 2^31 elements of h in float32, and planes of 9 GB between the backward pass's products: the last rows against the
    formula, and weight gradients that only they contribute to."""
    from diffputer_amd.gated import gated_linear
    M, K, N, tail = 2_100_000, 16, 1032, 70
    x, wg, wu, bg, bu, dh = make(tail, K, N, "f32", seed=24)
    ref = Ref(x, wg, wu, bg, bu, dh, "silu")
    big = torch.full((M, K), 0.5, device=DEV)
    big[-tail:] = x.to(DEV)
    leaves = [big.requires_grad_(), *[t.to(DEV).requires_grad_() for t in (wg, wu, bg, bu)]]
    h = gated_linear(*leaves)
    assert h.numel() > 1 << 31
    close(h[-tail:], ref.h, ref.eh, "h")
    assert torch.equal(h[:1000], h[:1].expand(1000, N)) and torch.equal(h[M // 2:M // 2 + 1000], h[:1].expand(1000, N))
    d = torch.zeros((M, N), device=DEV)
    d[-tail:] = dh.to(DEV)
    grads = torch.autograd.grad(h, leaves, d)
    close(grads[0][-tail:], ref.dx, ref.edx, "dx")
    assert not grads[0][:-tail].any()
    for name, g in zip(("wg", "wu", "bg", "bu"), grads[1:]):
        # sums of M terms, all but `tail` of them zero: the bound counts additions, of zeros too
        more = gamma(M) / gamma(tail)
        close(g, getattr(ref, "d" + name), more * getattr(ref, "ed" + name), "d" + name)
    del h, d, grads, big, leaves
    torch.cuda.empty_cache()


def test_bias_without_memory_is_refused():
    """A tensor that stands for others and has no memory of its own (a wrapper subclass) is no absent bias."""
    from diffputer_amd._lib import DiffputerError
    from diffputer_amd.gated import gated_linear

    class Wrapper(torch.Tensor):
        @staticmethod
        def __new__(cls, t):
            return torch.Tensor._make_wrapper_subclass(cls, t.shape, dtype=t.dtype, device=t.device)

        @classmethod
        def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
            raise NotImplementedError(func)

    x, w, b = torch.randn(3, 8, device=DEV), torch.randn(16, 8, device=DEV), torch.randn(16, device=DEV)
    for i in range(5):
        args = [x, w, w, b, b]
        args[i] = Wrapper(args[i])
        with pytest.raises((DiffputerError, RuntimeError), match="memory|null pointer"):
            gated_linear(*args)
    assert torch.isfinite(gated_linear(x, w, w, b, b)).all()


def test_backward_loses_no_tangent_and_no_trace():
    """A gradient that comes in with a tangent, or under a tracer, is refused as the forward call's arguments are."""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    from diffputer_amd._lib import DiffputerError
    from diffputer_amd.gated import gated_linear
    x, wg, wu, bg, bu, dh = [t.to(DEV) for t in make(9, 16, 8, "f32", seed=58)]
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    h = gated_linear(*leaves)
    want = torch.autograd.grad(h, leaves, dh, retain_graph=True)
    with forward_ad.dual_level():
        with pytest.raises((DiffputerError, RuntimeError), match="forward-mode"):
            torch.autograd.grad(h, leaves, forward_ad.make_dual(dh, torch.ones_like(dh)), retain_graph=True)
    with pytest.raises((DiffputerError, RuntimeError), match="traced"):
        make_fx(lambda d: torch.autograd.grad(h, leaves, d, retain_graph=True))(dh)
    got = torch.autograd.grad(h, leaves, dh)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

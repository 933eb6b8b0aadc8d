"""What the gated projection and the gradient clipping refuse, and what they do without a GPU (their C entry points check
every argument before the first HIP call)."""
import ctypes as C
import math
import sys

import pytest
import torch

from diffputer_amd import _lib
from diffputer_amd.gated import GatedLinear, gated_linear
from diffputer_amd.grads import clip_grads, grad_norm


def _err(lib):
    return lib.dp_last_error().decode()


def test_gated_linear_refuses():
    x, w, b = torch.randn(3, 4), torch.randn(5, 4), torch.randn(5)
    for args, kw, why in (
        ((x, w, w), {"act": "relu"}, "act must be"),
        ((x, w, w[:4]), {}, "expected"),
        ((x, w[:, :3], w[:, :3]), {}, "expected"),
        ((torch.randn(()), w, w), {}, "expected"),
        ((x, w[0], w[0]), {}, "expected"),
        ((x, w[:0], w[:0]), {}, "at least 1"),
        ((x[:, :0], w[:, :0], w[:, :0]), {}, "at least 1"),
        ((x, w, w, b[:4]), {}, "b_gate"),
        ((x, w, w, None, b.reshape(1, 5)), {}, "b_up"),
        ((x, w.bfloat16(), w), {}, "float32, or all bfloat16"),
        ((x.half(), w.half(), w.half()), {}, "float32, or all bfloat16"),
        ((x.double(), w.double(), w.double()), {}, "float32, or all bfloat16"),
        ((x, w, w, b.bfloat16()), {}, "b_gate"),
        ((x, w.to("meta"), w), {}, "is on meta"),
    ):
        with pytest.raises(ValueError, match=why):
            gated_linear(*args, **kw)
    with pytest.raises(_lib.DiffputerError, match="no CPU fallback"):
        gated_linear(x, w, w, b, b)


def test_grads_refuse():
    g = torch.randn(4)
    for call in (grad_norm, lambda t, **k: clip_grads(t, 1.0, **k)):
        with pytest.raises(_lib.DiffputerError, match="no CPU fallback"):
            call([g])
        with pytest.raises(ValueError, match="norm_type"):
            call([g], norm_type=1.0)
        with pytest.raises(ValueError, match="no tensors"):
            call([])
        with pytest.raises(ValueError, match="float16"):
            call([g.half()])
        with pytest.raises(ValueError, match="tensor 1 is on meta"):
            call([g, g.to("meta")])
    for limit in (-1.0, math.nan, "x"):
        with pytest.raises(ValueError):
            clip_grads([g], limit)


class _Binding:
    """Stands for csrc/dp_torch.so on the CPU: what clip_grads hands over, checked as the library checks it."""

    @staticmethod
    def grads(tensors, kind, limit):
        for i, t in enumerate(tensors):
            if not t.is_contiguous():
                return i
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors if t.numel())
        if limit is not None and any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise _lib.DiffputerError("two of the tensors share memory")
        norm = torch.stack([t.float().square().sum() for t in tensors]).sum().sqrt()
        if limit is not None:
            for t in tensors:
                t.mul_(min(1.0, limit / (float(norm) + 1e-6)))
        return norm


def _strided(base, size, stride, offset=0):
    return torch.as_strided(base, size, stride, offset)


def test_overlaps_of_tensors_with_gaps_are_refused(monkeypatch):
    """clip_grads refuses tensors that share memory, also where they are not dense and would be scaled as copies."""
    monkeypatch.setattr(_lib, "torch_side", lambda: _Binding)
    a, b = torch.arange(1.0, 41).reshape(5, 8), torch.arange(1.0, 41).reshape(5, 8)
    keep = a.clone()
    flat = a.view(-1)
    for ts in ([a[:, :3], a[:, :3]], [a[:, :3], a[:, 2:5]], [a[:, :3], a[:, 1:]], [flat[16:24], a[:, :2]], [a[:, :2], flat[16:24]], [b[:, :2], a[:, 1:4], b[:, 4:], a[:, 3:5]],
               [a[:, ::2], a[:, 4:5]], [a[::2, ::2], a[2:3]], [a, a[:, :2]], [a.t()[:3], a[:, 2:]], [a[:, 3], a[2]], [a[:, :2], a.view(torch.bfloat16)[:, 3:5]]):
        with pytest.raises(_lib.DiffputerError, match="share memory"):
            clip_grads(ts, 1.0)
        assert torch.equal(a, keep)
        assert abs(float(grad_norm(ts)) - math.sqrt(sum(float(t.double().square().sum()) for t in ts))) < 1e-3 * float(grad_norm(ts))      # reading twice is fine
    for t in (_strided(flat, (3, 2), (1, 1)), _strided(flat, (4, 3), (2, 1)), _strided(flat, (3, 5), (4, 2)), _strided(flat, (2, 3, 4), (1, 2, 3)), a[:, :1].expand(5, 4)):
        with pytest.raises(ValueError, match="share memory"):
            clip_grads([torch.ones(3), t], 1.0)
        assert torch.equal(a, keep)
    for ts in ([a[:, :3], a[:, 3:]], [a[:, ::2], a[:, 1::2]], [a[:, :2], a[:, 4:6], a[:, 2:4], a[:, 6:]], [a[::2], a[1::2, :5], a[1::2, 5:]], [a.t()[:3], a.t()[3:]], [flat[:8], a[1:, :2], a[1:, 2:]],
               [_strided(flat, (2, 3), (3, 2)), flat[10:12]], [a[:, :1], torch.ones(0), a[:, 1:3]], [a[:, :2], a.view(torch.bfloat16)[:, 4:6]]):
        a.copy_(keep)
        want = [t.clone() for t in ts]
        norm = clip_grads(ts, 1.0)
        for t, w in zip(ts, want):
            assert torch.allclose(t, w * min(1.0, 1.0 / (float(norm) + 1e-6)), rtol=2e-2 if t.dtype == torch.bfloat16 else 1e-5)
    a.copy_(keep)


def test_overlaps_against_enumeration():
    """The host's answer against all addresses of small tensors."""
    import random

    from diffputer_amd import grads
    r = random.Random(5)
    base = torch.zeros(4000)
    seen = [0, 0, 0, 0]

    def some():
        n = r.randint(1, 4)
        return _strided(base, [r.randint(1, 4) for _ in range(n)], [r.choice([1, 2, 3, 4, 5, 7, 8, 12, 16, 30, 60]) for _ in range(n)], r.randint(0, 60))

    def places(t):
        where = torch.zeros(1, dtype=torch.int64)
        for n, s in zip(t.shape, t.stride()):
            where = (where[:, None] + torch.arange(n) * s).reshape(-1)
        return (where + t.storage_offset()).tolist()

    for _ in range(3000):
        t, u = some(), some()
        p, q = places(t), places(u)
        for v, w in ((t, p), (u, q)):
            assert grads._meets_itself(v) == (len(set(w)) < len(w)), (v.shape, v.stride())
            seen[len(set(w)) < len(w)] += 1
        assert grads._meet(t, u) == bool(set(p) & set(q)), (t.shape, t.stride(), t.storage_offset(), u.shape, u.stride(), u.storage_offset())
        seen[2 + bool(set(p) & set(q))] += 1
    assert min(seen) > 300
    for _ in range(1500):
        pitch = r.choice([6, 8, 15])
        ts = [_strided(base, (r.randint(2, 4), r.randint(1, 3)), (pitch, r.choice([1, 2])), r.randint(0, 20)) for _ in range(r.randint(2, 5))]
        if any(grads._meets_itself(t) for t in ts):
            continue
        all_ = [x for t in ts for x in places(t)]
        try:
            grads._refuse_shared(ts, "x")
            assert len(set(all_)) == len(all_)
        except _lib.DiffputerError:
            assert len(set(all_)) < len(all_)


def test_many_views_of_one_table(monkeypatch):
    """Column ranges of one table are told apart without a look at every pair; one that meets another is found."""
    from diffputer_amd import grads
    pairs, meet = [], grads._meet
    monkeypatch.setattr(grads, "_meet", lambda o, t: pairs.append(1) or meet(o, t))
    a = torch.zeros(40, 1200)
    views = [a[:, 3 * i:3 * i + 3] for i in range(400)]
    rows = [a[i::7, ::2] for i in range(7)] + [a[i::7, 1::2] for i in range(7)]
    grads._refuse_shared(views, "x")
    grads._refuse_shared(views[::-1] + [torch.zeros(3, 4)[:, :2]], "x")
    assert not pairs
    grads._refuse_shared(rows, "x")
    assert pairs
    for more in (a[5:9, 1100:1102], a[::2, 7:8], a.view(-1)[17:18], a[:, 1199:]):
        with pytest.raises(_lib.DiffputerError, match="share memory"):
            grads._refuse_shared([*views, more], "x")
    # a range that wraps round the end of the table's row, beside one that it meets and one that it does not
    flat = a.view(-1)
    wrap = _strided(flat, (39, 4), (1200, 1), 1198)
    grads._refuse_shared([wrap, a[:, 2:1198]], "x")
    with pytest.raises(_lib.DiffputerError, match="share memory"):
        grads._refuse_shared([wrap, a[:, 1:5]], "x")
    with pytest.raises(_lib.DiffputerError, match="share memory"):
        grads._refuse_shared([wrap, a[:, 1199:]], "x")


def _calls():
    """Every entry point that takes tensors, as a function of one tensor (on the CPU: what is refused is refused before the device)."""
    w = torch.randn(5, 4)
    return [lambda t: gated_linear(t, w, w), lambda t: gated_linear(w[:3], t.expand(5, 4), w), lambda t: gated_linear(w, w, w, t[0, :1].expand(5)),
            lambda t: gated_linear(w, w, w, None, t[0, :1].expand(5)), lambda t: grad_norm([w, t]), lambda t: clip_grads([w, t], 1.0)]


@pytest.mark.parametrize("i", range(6))
def test_tangents_are_refused(i):
    """Forward-mode derivatives would be dropped without a word: a dual tensor is refused wherever it comes in."""
    from torch.autograd import forward_ad
    call, x = _calls()[i], torch.randn(1, 4)
    with forward_ad.dual_level():
        for grad in (False, True):
            base = x.clone().requires_grad_(grad)
            with pytest.raises(_lib.DiffputerError, match="forward-mode"):
                call(forward_ad.make_dual(base, torch.ones_like(x)))
            with torch.no_grad(), pytest.raises(_lib.DiffputerError, match="forward-mode"):
                call(forward_ad.make_dual(base, torch.ones_like(x)))
        with pytest.raises(_lib.DiffputerError, match="no CPU fallback"):
            call(x)                                                  # no tangent: as ever


@pytest.mark.parametrize("i", range(6))
@pytest.mark.parametrize("how", ["jit", "make_fx", "make_fx_symbolic", "make_fx_pre_dispatch", "fake"])
def test_traces_are_refused(how, i):
    """A trace would record the output's allocation and nothing that fills it."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    call, x = _calls()[i], torch.randn(1, 4)
    run = {"jit": lambda: torch.jit.trace(call, (x,)), "make_fx": lambda: make_fx(call)(x), "make_fx_symbolic": lambda: make_fx(call, tracing_mode="symbolic", _allow_non_fake_inputs=True)(x),
           "make_fx_pre_dispatch": lambda: make_fx(call, pre_dispatch=True)(x)}
    with pytest.raises(_lib.DiffputerError, match="traced"):
        if how == "fake":
            with FakeTensorMode(allow_non_fake_inputs=True) as mode:
                call(mode.from_tensor(x))
        else:
            run[how]()
    with pytest.raises(_lib.DiffputerError, match="no CPU fallback"):
        call(x)


def test_module_on_the_cpu():
    torch.manual_seed(1)
    for act, f in (("silu", torch.nn.functional.silu), ("gelu", torch.nn.functional.gelu), ("none", lambda t: t)):
        m = GatedLinear(7, 5, act=act)
        assert sorted(m.state_dict()) == ["gate.bias", "gate.weight", "up.bias", "up.weight"]
        x = torch.randn(2, 3, 7)
        assert torch.allclose(m(x), f(m.gate(x)) * m.up(x))
    assert GatedLinear(7, 5, bias=False).gate.bias is None
    with pytest.raises(ValueError):
        GatedLinear(7, 5, act="tanh")


def test_m_step_limit_on_the_cpu():
    from diffputer_amd import em
    X = torch.randn(40, 3)
    with pytest.raises(ValueError):
        em.m_step(X, 8, max_epochs=1, max_grad_norm=-1.0)
    torch.manual_seed(0)
    model, best = em.m_step(X, 8, max_epochs=2, max_grad_norm=1e-3)
    assert math.isfinite(best)


def test_build_takes_its_argument():
    """build(force=True) is how a rebuild was asked for; it is one of build()'s calls still."""
    import inspect

    import __graft_entry__ as entry
    for args in ({}, {"force": True}, {"force": False}):
        inspect.signature(entry.build).bind(**args)


FAKE = 1 << 12                                                     # an aligned address that nothing reads: every call below is refused first


def _fwd(lib, dtype=1, x=FAKE, ldx=64, wg=FAKE, wu=FAKE, ldw=64, bg=None, bu=None, h=FAKE, ldh=32, pre=None, M=10, N=32, K=64, act=1, ws=FAKE, ws_bytes=1 << 40):
    return lib.dp_gated_linear(dtype, x, ldx, wg, wu, ldw, bg, bu, h, ldh, pre, M, N, K, act, ws, ws_bytes, None)


def _bwd(lib, dtype=1, x=FAKE, ldx=64, wg=FAKE, wu=FAKE, ldw=64, pre=FAKE, dh=FAKE, lddh=32, dx=FAKE, dwg=FAKE, dwu=FAKE, dbg=None, dbu=None, M=10, N=32, K=64, act=1,
         ws=FAKE, ws_bytes=1 << 40):
    return lib.dp_gated_linear_bwd(dtype, x, ldx, wg, wu, ldw, pre, dh, lddh, dx, dwg, dwu, dbg, dbu, M, N, K, act, ws, ws_bytes, None)


@pytest.mark.parametrize("call", [_fwd, _bwd])
def test_c_entry_refuses(call):
    lib = _lib.load()
    bad = [dict(dtype=2), dict(dtype=-1), dict(M=-1), dict(M=1 << 29), dict(N=0), dict(K=0), dict(N=-5), dict(N=(1 << 20) + 1), dict(K=(1 << 20) + 1), dict(act=3), dict(act=-1),
           dict(x=None), dict(wg=None), dict(wu=None), dict(ldx=63), dict(ldw=63), dict(x=FAKE + 1), dict(wg=FAKE + 1), dict(dtype=0, wu=FAKE + 2)]
    bad += [dict(h=None), dict(ldh=31), dict(h=FAKE + 1), dict(bg=FAKE + 1), dict(pre=FAKE + 8)] if call is _fwd else \
           [dict(pre=None), dict(dh=None), dict(lddh=31), dict(dh=FAKE + 1), dict(pre=FAKE + 8), dict(dx=FAKE + 1), dict(dwg=FAKE + 1), dict(dbu=FAKE + 1)]
    for kw in bad:
        assert call(lib, **kw) == -1, kw                            # DP_EINVAL
        assert "dp_gated_linear" in _err(lib), kw
    for kw in (dict(ws=None), dict(ws_bytes=0), dict(ws=FAKE + 128)):
        assert call(lib, **kw) == -4, kw                            # DP_EWORKSPACE
    assert _fwd(lib, M=0, x=None, h=None, ws=None) == 0             # no rows: nothing to do


def test_gated_sizes():
    lib = _lib.load()
    assert lib.dp_gated_linear_pre_bytes(0, 10, 33) == 10 * 2 * 36 * 4
    assert lib.dp_gated_linear_pre_bytes(1, 10, 33) == 10 * 2 * 36 * 5 // 2
    assert lib.dp_gated_linear_pre_bytes(0, -1, 33) == 0 and lib.dp_gated_linear_pre_bytes(0, 5, 0) == 0 and lib.dp_gated_linear_pre_bytes(2, 5, 5) == 0

    def ws(dtype, M, N, K, backward, at=FAKE):
        return lib.dp_gated_linear_workspace_bytes(dtype, at, K, at, at, K, M, N, K, backward)

    for args in ((2, 5, 5, 5, 0), (0, -1, 5, 5, 0), (0, 5, 0, 5, 1), (0, 5, 5, 0, 1)):
        assert ws(*args) == 0
    for dtype in (0, 1):
        for M, N, K in ((0, 5, 5), (1, 1, 1), (1, 2048, 1024), (24, 8192, 4096), (16384, 64, 9), (4096, 2048, 1024), ((1 << 29) - 1, 64, 64)):
            for backward in (0, 1):
                assert ws(dtype, M, N, K, backward) >= 256
    assert ws(0, 10, 10, 10, 16) == 0 and ws(0, 10, 10, 10, -1) == 0
    for grads in range(1, 16):
        assert ws(1, 300, 200, 100, grads) >= 2 * 300 * 256 * 2
    # a float32 plane of a large batch passes 32 bits
    assert ws(0, 1 << 20, 4096, 64, 1) >= 2 * (1 << 20) * 4096 * 4
    # rows that are not aligned are copied: x and both weights
    assert ws(1, 4096, 2048, 1024, 0, FAKE + 2) >= (4096 + 2 * 2048) * 1024 * 2 > ws(1, 4096, 2048, 1024, 0)
    assert lib.dp_gated_linear_pre_bytes(0, 1 << 20, 4096) == 2 * (1 << 20) * 4096 * 4


@pytest.fixture
def tune():
    lib = _lib.load()

    def put(kernel, splits=0):
        _lib.check(lib.dp_tune(b"gated_kernel", kernel), "dp_tune")
        _lib.check(lib.dp_tune(b"gated_splits", splits), "dp_tune")

    yield put
    put(0)


def _plan(dtype, M, N, K, grads, at=FAKE):
    k = (C.c_int * 3)()
    assert _lib.load().dp_gated_linear_plan(dtype, at, K, at, at, K, M, N, K, grads, k) == 0, _err(_lib.load())
    return list(k)


DX, DWG, DWU, DB = 1, 2, 4, 8


@pytest.mark.parametrize("kernel", [0, 1, 128, 256])
@pytest.mark.parametrize("M,N,K", [(1 << 28, 8, 136), ((1 << 29) - 1, 8, 8), (1 << 28, 136, 8), ((1 << 29) - 1, 8, 200), ((1 << 29) - 1, 1 << 20, 1 << 20), (1 << 20, 1 << 18, 1 << 18),
                                   (4096, 2048, 1024), (1537, 1203, 777), (100, 64, 9), (1, 8, 8)])
def test_planes_are_of_the_type_that_their_reader_takes(tune, kernel, M, N, K):
    """The general kernel (1) reads dg and du as float32, the tile kernels in the layer's own type: also where a tile kernel's grid
    would not fit (2^22 workgroups), a choice that the largest layers come to."""
    tune(kernel)
    for at in (FAKE, FAKE + 2):
        for grads in range(1, 16):
            dx, dw, plane = _plan(1, M, N, K, grads, at)
            assert (dx == -1) == (not grads & DX) and (dw == -1) == (not grads & (DWG | DWU))
            for k in (dx, dw):
                assert k in (-1, 1, 128, 256)
                assert k != 1 or plane == 0, (M, N, K, grads, dx, dw, plane)
                assert k < 64 or plane == 1, (M, N, K, grads, dx, dw, plane)


def test_large_layers_keep_tile_kernels():
    """Where the cheaper tile's grid does not fit, the other tile's does."""
    assert _plan(1, 1 << 28, 8, 136, DX)[0] == 256
    assert _plan(1, (1 << 29) - 1, 8, 8, DX | DWG | DWU)[0] == 256
    assert _plan(1, 4096, 2048, 1024, DX | DWG | DWU) == [128, 128, 1]
    assert _plan(1, 32768, 2048, 2048, 0)[0] == 256 and _plan(1, 1, 2048, 1024, 0)[0] == 2 and _plan(0, 1, 2048, 1024, 0) == [2, -1, -1]


def test_settings_that_change_during_a_call(tune):
    """A thread changes the tuning knobs while another plans calls: every plan and workspace is one that some setting gives, and none of
    them is kept for another setting."""
    import threading
    lib = _lib.load()
    settings = [(k, s) for k in (0, 1, 128, 256) for s in (0, 5)]
    sizes = [(100 + 37 * i, 64 + 40 * (i % 11), 64 + 24 * (i % 17), at) for i in range(90) for at in (FAKE, FAKE + 2)]

    def query(M, N, K, at):
        k = (C.c_int * 3)()
        lib.dp_gated_linear_plan(1, at, K, at, at, K, M, N, K, DX | DWG | DWU, k)
        return tuple(k)

    def workspace(M, N, K, at):
        return tuple(lib.dp_gated_linear_workspace_bytes(1, at, K, at, at, K, M, N, K, g) for g in (0, DX | DWG | DWU))

    plans, spaces = {}, {}
    for t in settings:
        tune(*t)
        for z in sizes:
            plans.setdefault(z, set()).add(query(*z))
            for i, b in enumerate(workspace(*z)):
                spaces.setdefault((z, i), set()).add(b)
    tune(0)
    serial = {z: (query(*z), workspace(*z)) for z in sizes}
    stop, n = threading.Event(), [0]

    def change():
        while not stop.is_set():
            for k, s in settings:
                lib.dp_tune(b"gated_kernel", k)
                lib.dp_tune(b"gated_splits", s)
            n[0] += 1

    t = threading.Thread(target=change)
    interval = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)                                    # so that both threads are inside the library most of the time
    t.start()
    try:
        for _ in range(150):
            for z in sizes:
                assert query(*z) in plans[z], z
                for i, b in enumerate(workspace(*z)):
                    assert b in spaces[z, i], (z, i)
    finally:
        stop.set()
        t.join()
        sys.setswitchinterval(interval)
    assert n[0] > 100
    tune(0)
    assert {z: (query(*z), workspace(*z)) for z in sizes} == serial


def test_plan_refuses():
    lib = _lib.load()
    k = (C.c_int * 3)()
    for args in ((2, FAKE, 8, FAKE, FAKE, 8, 5, 8, 8, 0, k), (1, FAKE, 8, FAKE, FAKE, 8, -1, 8, 8, 0, k), (1, FAKE, 8, FAKE, FAKE, 8, 5, 8, 8, 16, k), (1, FAKE, 8, FAKE, FAKE, 8, 5, 8, 8, 0, None)):
        assert lib.dp_gated_linear_plan(*args) == -1 and "dp_gated_linear_plan" in _err(lib)
    assert _plan(1, 0, 8, 8, 1) == [-1, -1, -1]


def _table(ptrs, numel, dtypes):
    n = len(ptrs)
    return n, (C.c_void_p * n)(*ptrs), (C.c_int64 * n)(*numel), (C.c_int * n)(*dtypes)


def test_c_clip_refuses():
    lib = _lib.load()
    big = 1 << 30

    def clip(ptrs=(FAKE,), numel=(8,), dtypes=(0,), kind=2, limit=1.0, norm=FAKE, ws=FAKE, ws_bytes=big, n=None):
        t = _table(ptrs, numel, dtypes)
        return lib.dp_clip_grads(t[0] if n is None else n, *t[1:], kind, limit, norm, ws, ws_bytes, None)

    def norm_(ptrs=(FAKE,), numel=(8,), dtypes=(0,), kind=2, norm=FAKE, ws=FAKE, ws_bytes=big, n=None):
        t = _table(ptrs, numel, dtypes)
        return lib.dp_grad_norm(t[0] if n is None else n, *t[1:], kind, norm, ws, ws_bytes, None)

    for call, name in ((clip, "dp_clip_grads"), (norm_, "dp_grad_norm")):
        for kw in (dict(dtypes=(5,)), dict(numel=(-1,)), dict(numel=(1 << 60,)), dict(ptrs=(None,)), dict(ptrs=(FAKE + 2,)), dict(ptrs=(FAKE + 1,), dtypes=(1,)),
                   dict(kind=1), dict(norm=None), dict(n=-1)):
            assert call(**kw) == -1, (name, kw)
            assert name in _err(lib)
        for kw in (dict(ws=None), dict(ws_bytes=8), dict(ws=FAKE + 4)):
            assert call(**kw) == -4, (name, kw)
    for limit in (-0.5, math.nan):
        assert clip(limit=limit) == -1
    for ptrs, numel, dtypes in (((FAKE, FAKE), (8, 8), (0, 0)), ((FAKE, FAKE + 28), (8, 8), (0, 1)), ((FAKE + 64, FAKE), (4, 17), (0, 0)),
                                ((FAKE, FAKE + 4, FAKE + 8), (100, 0, 1), (0, 0, 0))):
        assert clip(ptrs=ptrs, numel=numel, dtypes=dtypes) == -1 and "share memory" in _err(lib)

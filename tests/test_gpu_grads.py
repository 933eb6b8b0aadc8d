"""The global gradient norm and clipping (`diffputer_amd.grads`, dp_grad_norm / dp_clip_grads) on the GPU against float64.

Tolerances: the sum of squares is float64 (relative error n 2^-53, nothing here), its root is rounded to float32 once: 2^-24,
held to 2^-23.  A clipped element is g c: c is rounded to float32 (2^-24), the product once more (2^-24) and then to the
tensor's type (eps / 2)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float64


def tensors(sizes, dtypes, seed=0, scale=1e-2):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(*(s if isinstance(s, tuple) else (s,)), generator=gen) * scale * (1 + i % 5)).to(dtypes[i % len(dtypes)]).to(DEV)
            for i, s in enumerate(sizes)]


def norm_of(grads, kind=2.0):
    flat = torch.cat([g.detach().cpu().to(F8).reshape(-1) for g in grads])
    return float(flat.square().sum().sqrt()) if kind == 2.0 else float(flat.abs().max()) if flat.numel() else 0.0


def check(grads, limit, kind=2.0):
    from diffputer_amd.grads import clip_grads, grad_norm
    before = [g.detach().cpu().to(F8).clone() for g in grads]
    norm = norm_of(grads, kind)
    for got in (grad_norm(grads, kind), clip_grads(grads, limit, kind)):
        assert got.shape == () and got.dtype == torch.float32 and got.is_cuda
        assert abs(float(got) - norm) <= 2.0 ** -23 * norm + 1e-45, (float(got), norm)
    coef = min(1.0, limit / (norm + 1e-6))
    for b, g in zip(before, grads):
        want, got = b * coef, g.detach().cpu().to(F8)
        if coef == 1.0:
            assert torch.equal(got, b)
            continue
        tol = (torch.finfo(g.dtype).eps / 2 + 3 * 2.0 ** -24) * want.abs() * 1.01 + 1e-38
        assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())


F32, BF = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtypes", [[F32], [BF], [F32, BF]])
@pytest.mark.parametrize("sizes", [[1], [3], [7, 1, 2], [8192], [8193, 16385, 5], [(64, 9), (64,), (128, 64), (128,)], [100_003], [2_000_001, 333]])
def test_sizes_and_types(sizes, dtypes):
    for limit in (0.01, 1e9, 0.0):
        check(tensors(sizes, dtypes, seed=len(sizes)), limit)


@pytest.mark.parametrize("n", [159, 160, 161, 320, 401, 1000])
def test_many_tensors(n):
    check(tensors([(i * 37) % 1500 for i in range(n)], [F32, BF, BF], seed=n), 0.5)      # zero sizes among them


@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_norm_types(kind):
    check(tensors([1000, 77, (3, 5)], [F32, BF], seed=2), 0.003, kind)


def test_no_elements():
    from diffputer_amd.grads import clip_grads, grad_norm
    e = [torch.empty(0, device=DEV), torch.empty(3, 0, device=DEV, dtype=BF)]
    assert float(grad_norm(e)) == 0.0 and float(clip_grads(e, 1.0)) == 0.0


@pytest.mark.parametrize("dtype", [F32, BF])
def test_views_of_one_buffer_any_alignment(dtype):
    """Views that start at every element offset of a flat buffer; the elements between them stay as they were."""
    from diffputer_amd.grads import clip_grads
    buf = torch.full((60_000,), 3.0, dtype=dtype, device=DEV)
    views, at, used = [], 1, torch.zeros(60_000, dtype=torch.bool, device=DEV)
    for i in range(40):
        n = (i * 53) % 1400 + 1
        views.append(buf[at:at + n])
        used[at:at + n] = True
        at += n + 1 + i % 3
    norm = norm_of(views)
    clip_grads(views, norm / 4)
    assert bool((buf[~used] == 3.0).all())
    assert float((buf[used].to(F8) - 0.75).abs().max()) <= (torch.finfo(dtype).eps / 2 + 2.0 ** -22) * 0.75 + 0.75e-6
    whole = list(torch.full((1000,), 3.0, dtype=dtype, device=DEV).split([1, 2, 3, 4, 5, 985]))     # one behind the other
    check(whole, 1.0)


def test_extreme_values():
    """Squares that would overflow or vanish in float32 do neither."""
    check([torch.full((1000,), 1e25, device=DEV), torch.full((10,), -3e37, device=DEV)], 1.0)
    check([torch.full((1000,), 1e-30, device=DEV)], 1.0)
    check([torch.full((1000,), 1e30, device=DEV, dtype=BF)], 1e10)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_nan_and_inf(dtype, kind):
    from diffputer_amd.grads import clip_grads, grad_norm
    for bad in (math.nan, math.inf, -math.inf):
        for at in (0, 5, 99_999):
            g = tensors([100_000, 10], [dtype], seed=4)
            g[0][at] = bad
            norm = float(grad_norm(g, kind))
            assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
            before = [t.clone() for t in g]
            with pytest.raises(RuntimeError):
                clip_grads(g, 1.0, kind, error_if_nonfinite=True)
            assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(before, g))
            clip_grads(g, 1.0, kind)
            if math.isnan(bad):
                assert all(bool(torch.isnan(t).all()) for t in g)
            else:                                                   # the coefficient is 0: zeros, and inf * 0 = NaN
                assert bool(torch.isnan(g[0][at])) and float(g[1].abs().max()) == 0.0


def test_layouts():
    from diffputer_amd.grads import clip_grads, grad_norm
    base = torch.randn(40, 60, device=DEV)
    t, s = base.t(), torch.randn(30, 50, device=DEV)[:, ::2]       # transposed: dense; every other column: not
    p = torch.randn(4, 6, 5, device=DEV).permute(2, 0, 1)
    rest = s._base[:, 1::2].clone()
    check([t, s, p], 0.1)
    assert torch.equal(s._base[:, 1::2], rest)
    with pytest.raises(ValueError):
        clip_grads([torch.randn(1, 5, device=DEV).expand(4, 5)], 1.0)
    assert abs(float(grad_norm([torch.ones(1, 5, device=DEV).expand(4, 5)])) - math.sqrt(20)) < 1e-5


def test_shared_memory_is_refused():
    from diffputer_amd._lib import DiffputerError
    from diffputer_amd.grads import clip_grads, grad_norm
    g = torch.randn(1000, device=DEV)
    keep = g.clone()
    for pair in ([g, g], [g[:600], g[599:]], [g[500:], torch.randn(3, device=DEV), g[:501]]):
        with pytest.raises(DiffputerError, match="share memory"):
            clip_grads(pair, 0.1)
    assert torch.equal(g, keep)
    assert abs(float(grad_norm([g, g])) - norm_of([g, g])) <= 1e-5 * norm_of([g, g])       # reading it twice is fine


def test_more_than_32_bits_of_bytes():
    """A tensor of 4.8 GB (and odd ones beside it): every element once, none twice."""
    from diffputer_amd.grads import clip_grads
    n = 1_200_000_007
    g = [torch.full((n,), 2.0, device=DEV), torch.full((5,), 2.0, device=DEV), torch.full((3_000_001,), 2.0, dtype=BF, device=DEV)]
    count = sum(t.numel() for t in g)
    norm = float(clip_grads(g, math.sqrt(count)))                    # to a half, but for the 1e-6 and two roundings
    assert abs(norm - 2 * math.sqrt(count)) <= 2.0 ** -23 * norm
    for t in g:
        assert float(t.amin()) == float(t.amax())
        assert abs(float(t[-1]) - 1.0) <= torch.finfo(t.dtype).eps / 2 + 2.0 ** -21
    del g
    torch.cuda.empty_cache()


def test_same_bits_twice_and_within_the_limit():
    from diffputer_amd.grads import clip_grads
    one, two = tensors([999_999, 12345], [F32, BF], seed=6), tensors([999_999, 12345], [F32, BF], seed=6)
    a, b = clip_grads(one, 0.7), clip_grads(two, 0.7)
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(one, two))
    c = clip_grads(one, 0.71)                                       # now within: nothing moves
    assert abs(float(c) - 0.7) < 1e-3 and all(torch.equal(x, y) for x, y in zip(one, two))


def test_side_stream_and_capture():
    from diffputer_amd.grads import clip_grads
    src = [tensors([70_001, 33, 4096], [F32, BF], seed=s) for s in (7, 8)]
    want = []
    for g in src:
        c = [t.clone() for t in g]
        want.append((clip_grads(c, 0.05), c))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = [t.clone() for t in src[0]]
        n = clip_grads(c, 0.05)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(n, want[0][0]) and all(torch.equal(a, b) for a, b in zip(c, want[0][1]))
    static = [t.clone() for t in src[0]]
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            n = clip_grads(static, 0.05)
        graphs.append((graph, n))
    for it in range(6):
        for t, v in zip(static, src[it % 2]):
            t.copy_(v)
        graph, n = graphs[it % 2]
        graph.replay()
        clip_grads([torch.randn(50, device=DEV)], 1.0)
        torch.cuda.synchronize()
        assert torch.equal(n, want[it % 2][0]) and all(torch.equal(a, b) for a, b in zip(static, want[it % 2][1])), it


def test_m_step_clips():
    """em.m_step(max_grad_norm=...): every Adam step sees gradients within the limit, and without a limit nothing changes."""
    from diffputer_amd import em, grads
    seen, plain = [], em.clip_grads

    def spy(gs, limit, *a, **k):
        out = plain(gs, limit, *a, **k)
        seen.append((float(out), norm_of(gs)))
        return out

    X = torch.randn(300, 9, device=DEV)
    runs = []
    for limit in (None, 1e-3, None):
        torch.manual_seed(3)
        em.clip_grads = spy
        try:
            gen = torch.Generator(device=DEV).manual_seed(1)
            model, best = em.m_step(X, 64, max_epochs=4, batch_size=128, generator=gen, max_grad_norm=limit)
        finally:
            em.clip_grads = plain
        runs.append((model.state_dict(), best))
    assert len(seen) == 12 and all(before > 1e-3 and after <= 1e-3 * (1 + 1e-5) for before, after in seen)
    assert all(torch.equal(a, b) for a, b in zip(runs[0][0].values(), runs[2][0].values())) and math.isfinite(runs[1][1])
    assert grads.clip_grads is plain


def test_a_graph_that_kept_a_gradient_notices():
    """Clipping writes in place: a graph that saved the tensor before must not use it afterwards."""
    from diffputer_amd.grads import clip_grads, grad_norm
    g = torch.randn(100, device=DEV)
    w = torch.randn(100, device=DEV, requires_grad=True)
    y = (w * g).sum()
    grad_norm([g])
    z = (w * g).sum()
    torch.autograd.grad(y, w)
    clip_grads([g], 0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(z, w)
    with torch.inference_mode():
        g = torch.full((100,), 3.0, device=DEV)
        clip_grads([g], 1.0)
    # coefficient 1 / (30 + 1e-6) in float32, one product: 2^-23 of 0.1
    assert abs(float(g[0]) - 3.0 / (30.0 + 1e-6)) <= 2.0 ** -22 * 0.1


@pytest.mark.parametrize("dtype", [F32, BF])
def test_lazily_negated_tensors(dtype):
    """A tensor whose negation is a bit: scaled in place through the bit, and the memory behind it with it."""
    from diffputer_amd.grads import clip_grads, grad_norm
    base = torch.randn(1000, device=DEV).to(dtype)
    keep, lazy = base.clone(), torch._neg_view(base)
    other = torch.randn(77, device=DEV)
    norm = norm_of([keep, other])
    assert abs(float(grad_norm([lazy, other])) - norm) <= 2.0 ** -23 * norm
    want = [(-keep).clone(), other.clone()]
    clip_grads(want, 0.3)
    got = [lazy, other]
    n = clip_grads(got, 0.3)
    assert abs(float(n) - norm) <= 2.0 ** -23 * norm
    assert lazy.is_neg() and all(torch.equal(a.resolve_neg(), b) for a, b in zip(got, want))
    assert torch.equal(base, -want[0])


def test_shared_memory_of_tensors_with_gaps():
    """Overlaps of tensors that are not dense are refused before anything is scaled; views that interleave are scaled once each."""
    from diffputer_amd._lib import DiffputerError
    from diffputer_amd.grads import clip_grads
    a = torch.randn(300, 8, device=DEV)
    keep = a.clone()
    for ts in ([a[:, :3], a[:, :3]], [a[:, :3], a[:, 2:5]], [a[:, :3], a[:, 1:]], [a.view(-1)[16:24], a[:, :2]], [a, a[:, :2]], [a.t()[:3], a[:, 2:]]):
        with pytest.raises(DiffputerError, match="share memory"):
            clip_grads(ts, 0.1)
    with pytest.raises(ValueError, match="share memory"):
        clip_grads([torch.as_strided(a, (3, 2), (1, 1))], 0.1)
    assert torch.equal(a, keep)
    check([a[:, ::2], a[:, 1:4:2], a[:, 5::2]], 0.1)
    a.copy_(keep)
    check([a[:, :3], a[:, 3:], torch.randn(5, device=DEV)], 0.1)

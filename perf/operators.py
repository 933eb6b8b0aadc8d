"""Cases of the gated projection h = act(x Wg^T + bg) * (x Wu^T + bu) (forward, and forward with backward) and of the
clipping of many gradient tensors by their global norm.

`run` computes a case in plain torch operations, or, with `own` set, through diffputer_amd's HIP kernels."""
import math

import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    g = {"op": "gated", "act": "silu", "bias": True, "strided": False}
    c = {"op": "clip", "above": True}
    return [
        # one row through the denoiser's H -> 2H layer at H = 1024: a request of one row, where latency counts
        {"name": "gated_row1_bf16", **g, "dtype": "bf16", "train": False, "m": 1, "k": 1024, "n": 2048},
        # a handful of requests through a wide layer: bound by reading the weights
        {"name": "gated_rows24_bf16", **g, "dtype": "bf16", "train": False, "m": 24, "k": 4096, "n": 8192, "bias": False},
        # a small table's first layer: 9 columns (odd rows in memory) to H = 64
        {"name": "gated_table9_f32", **g, "dtype": "f32", "train": False, "m": 100, "k": 9, "n": 64},
        # the sampler's row chunk through a 2H -> 2H layer
        {"name": "gated_chunk_bf16", **g, "dtype": "bf16", "train": False, "m": 32768, "k": 2048, "n": 2048},
        # the M-step's batch of 4096 through H -> 2H, forward and backward, in both types
        {"name": "gated_train_bf16", **g, "dtype": "bf16", "train": True, "m": 4096, "k": 1024, "n": 2048},
        {"name": "gated_train_f32", **g, "dtype": "f32", "train": True, "m": 4096, "k": 1024, "n": 2048},
        # sizes that divide nothing, a column range of a wider table, the other activation
        {"name": "gated_ragged_bf16", **g, "dtype": "bf16", "train": True, "m": 1537, "k": 777, "n": 1203, "act": "gelu", "strided": True},
        # a wide block trained on many rows: the largest
        {"name": "gated_train_large", **g, "dtype": "bf16", "train": True, "m": 16384, "k": 4096, "n": 8192, "bias": False},
        # the gradients of a small denoiser (9 columns, H = 64): latency
        {"name": "clip_h64", **c, "shapes": "denoiser", "dtype": "f32", "d_in": 9, "hid": 64},
        # the gradients of the M-step's denoiser at H = 1024
        {"name": "clip_h1024", **c, "shapes": "denoiser", "dtype": "f32", "d_in": 9, "hid": 1024},
        # many tensors of odd sizes in one flat buffer, as gradient buckets hold them
        {"name": "clip_bucket_bf16", **c, "shapes": "bucket", "dtype": "bf16", "tensors": 301, "total": 1 << 27},
        # a large set that is within the limit: only the norm has to be found
        {"name": "clip_within_f32", **c, "shapes": "bucket", "dtype": "f32", "tensors": 37, "total": 200_000_003, "above": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.65:
        dtype, train = rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.6
        case = {"op": "gated", "act": rng.choice(["silu", "silu", "gelu"]), "bias": rng.random() < 0.6, "strided": rng.random() < 0.3,
                "dtype": dtype, "train": train}
        most = 4e9 * (100 if dtype == "bf16" else 10)               # products of one pass: a tenth of it in float32
        while True:
            m, k, n = _log(rng, 1, 16384), _log(rng, 8, 4096), _log(rng, 8, 8192)
            if rng.random() < 0.5:                                   # widths are often whole multiples, and often not
                k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
            if m * k * n <= most:
                return {**case, "m": m, "k": k, "n": n}
    dtype, above = rng.choice(["bf16", "f32"]), rng.random() < 0.7
    if rng.random() < 0.4:
        return {"op": "clip", "above": above, "shapes": "denoiser", "dtype": "f32", "d_in": _log(rng, 3, 300), "hid": 64 * _log(rng, 1, 24)}
    tensors = _log(rng, 1, 400)
    return {"op": "clip", "above": above, "shapes": "bucket", "dtype": dtype, "tensors": tensors, "total": max(tensors, _log(rng, 1000, 200_000_000))}


# ---- inputs -------------------------------------------------------------------------------------------------------
def _clip_sizes(case):
    """[(shape)] of the gradients: the denoiser's 14 tensors, or `tensors` vectors whose uneven lengths add up to `total`."""
    if case["shapes"] == "denoiser":
        d, h = case["d_in"], case["hid"]
        pairs = [(h, d), (2 * h, h), (2 * h, 2 * h), (h, 2 * h), (d, h), (h, h), (h, h)]
        return [s for o, i in pairs for s in ((o, i), (o,))]
    t, total = case["tensors"], case["total"]
    weight = [1.0 + (7 * i % 13) for i in range(t)]                   # lengths that differ by up to 13 times
    sizes = [max(1, int((total - t) * w / sum(weight))) for w in weight]
    sizes[-1] += max(0, total - sum(sizes))
    return [(s,) for s in sizes]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] == "clip":
        shapes = _clip_sizes(case)
        count = [math.prod(s) for s in shapes]
        flat = torch.randn(sum(count), device=DEV, generator=gen).mul_(1e-3)
        if case["shapes"] == "denoiser":
            grads = [p.reshape(s).clone() for p, s in zip(flat.split(count), shapes)]     # every parameter's own .grad
            back = grads
        else:
            flat = flat.to(dt)
            grads, back = list(flat.split(count)), flat               # views of one buffer: their starts have any alignment
        norm = 1e-3 * math.sqrt(sum(count))                           # about what the norm is
        # the limit is a schedule that falls with every pass: in-place clipping then has something to clip in each
        return {"op": "clip", "grads": grads, "back": back, "limit": norm * (0.37 if case["above"] else 1e6), "above": case["above"]}
    m, k, n = case["m"], case["k"], case["n"]

    def rnd(*shape):
        return torch.randn(*shape, device=DEV, generator=gen)

    def uni(*shape):
        return (torch.rand(*shape, device=DEV, generator=gen) * 2 - 1).mul_(1 / math.sqrt(k))

    x = rnd(m, k + 13).to(dt)[:, 5:5 + k] if case["strided"] else rnd(m, k).to(dt)
    w = [uni(n, k).to(dt) for _ in range(2)]
    b = [uni(n).to(dt) for _ in range(2)] if case["bias"] else [None, None]
    s = {"op": "gated", "act": case["act"], "train": case["train"], "x": x, "wg": w[0], "wu": w[1], "bg": b[0], "bu": b[1]}
    if case["train"]:
        s["dh"] = rnd(m, n).mul_(1e-2).to(dt)
        for name in ("x", "wg", "wu", "bg", "bu"):
            if s[name] is not None:
                s[name] = s[name].detach().requires_grad_()
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------
def _plain_act(g, act):
    """act(g) and act'(g)"""
    if act == "silu":
        s = 1 / (1 + torch.exp(-g))
        return g * s, s * (1 + g * (1 - s))
    c = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
    return g * c, c + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))


@torch.no_grad()
def _plain_gated(s):
    dt = s["x"].dtype
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    if s["bg"] is not None:
        g, u = g + s["bg"].float(), u + s["bu"].float()
    a, da = _plain_act(g, s["act"])
    out = {"h": (a * u).to(dt)}
    if s["train"]:
        dh = s["dh"].float()
        du, dg = dh * a, dh * u * da
        out["dx"] = (dg @ wg + du @ wu).to(dt)
        out["dwg"], out["dwu"] = (dg.t() @ x).to(dt), (du.t() @ x).to(dt)
        if s["bg"] is not None:
            out["dbg"], out["dbu"] = dg.sum(0, dtype=torch.float64).to(dt), du.sum(0, dtype=torch.float64).to(dt)
    return out


@torch.no_grad()
def _plain_clip(grads, limit):
    norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt()
    coef = (limit / (norm + 1e-6)).clamp(max=1.0).float()
    for g in grads:
        g.copy_(g.float() * coef)
    return norm.float()


def run(state):
    if state["op"] == "clip":
        limit = state["limit"]
        if state["above"]:
            state["limit"] *= 0.9999
        if own:
            from diffputer_amd.grads import clip_grads
            norm = clip_grads(state["grads"], limit)
        else:
            norm = _plain_clip(state["grads"], limit)
        return {"norm": norm, "grads": state["back"]}
    if not own:
        return _plain_gated(state)
    from diffputer_amd.gated import gated_linear
    args = [state[name] for name in ("x", "wg", "wu", "bg", "bu")]
    if not state["train"]:
        with torch.no_grad():
            return {"h": gated_linear(*args, act=state["act"])}
    h = gated_linear(*args, act=state["act"])
    leaves = [name for name in ("x", "wg", "wu", "bg", "bu") if state[name] is not None]
    grads = torch.autograd.grad(h, [state[name] for name in leaves], state["dh"])
    return {"h": h.detach(), **{"d" + name: g for name, g in zip(leaves, grads)}}


# ---- what a pass cannot do without, and what it should give ---------------------------------------------------------
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "clip":
        count = sum(math.prod(s) for s in _clip_sizes(case))
        # within the limit the gradients stay as they are: they are read, and nothing is written
        return {"bytes": e * count * (2 if case["above"] else 1) + 4, "flops": count * (3 if case["above"] else 2)}
    m, k, n = case["m"], case["k"], case["n"]
    weights = 2 * n * k + (2 * n if case["bias"] else 0)
    if not case["train"]:
        return {"bytes": e * (m * k + weights + m * n), "flops": 4 * m * n * k}
    return {"bytes": e * (2 * m * k + 2 * weights + 2 * m * n), "flops": 12 * m * n * k}


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "clip":
        total = torch.zeros((), dtype=f8, device=DEV)
        for g in s["grads"]:
            total += torch.linalg.vector_norm(g.to(f8)) ** 2
        norm = torch.sqrt(total)
        scale = torch.minimum(torch.ones_like(norm), s["limit"] / (norm + 1e-6))
        back = [g.to(f8) * scale for g in s["back"]] if isinstance(s["back"], list) else s["back"].to(f8) * scale
        return {"norm": norm, "grads": back}
    x, wg, wu = (s[k].detach().to(f8) for k in ("x", "wg", "wu"))
    zero = torch.zeros(case["n"], dtype=f8, device=DEV)
    bg, bu = (zero if s[k] is None else s[k].detach().to(f8) for k in ("bg", "bu"))
    gate, up = torch.addmm(bg, x, wg.t()), torch.addmm(bu, x, wu.t())
    if case["act"] == "silu":
        cdf = torch.sigmoid(gate)
        slope = cdf + gate * torch.sigmoid(-gate) * cdf
    else:
        cdf = torch.special.ndtr(gate)
        slope = cdf + gate * torch.exp(-gate ** 2 / 2) / math.sqrt(2 * math.pi)
    res = {"h": gate * cdf * up}
    if case["train"]:
        d = s["dh"].to(f8)
        d_up = d * gate * cdf
        d_gate = d * up * slope
        res["dx"] = torch.mm(d_gate, wg) + torch.mm(d_up, wu)
        res["dwg"] = torch.mm(x.t(), d_gate).t()
        res["dwu"] = torch.mm(x.t(), d_up).t()
        if case["bias"]:
            res["dbg"] = torch.sum(d_gate, 0)
            res["dbu"] = torch.sum(d_up, 0)
    return res

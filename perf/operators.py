"""What is measured of the norm, the 8-bit product and the gradient clipping: cases, inputs, one pass, its work, its exact result.

Four kinds of case:

``norm``       root-mean-square norm behind the residual's addition as a training step uses it: forward and backward.
``norm_fp8``   the same norm as serving uses it: the output in e4m3 with one scale per row and block of 128 channels.
``mix_fp8``    ``y = x @ w^T + bias`` of e4m3 rows (a scale per row and 128 channels) and e4m3 weights (a scale per 128 x 128).
``clip``       the global norm of many gradient tensors and their clipping.

With ``own`` true a pass calls the package; otherwise it computes the same in elementary torch operations, in 32 bits (sums of
whole gradients in 64).
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
BLOCK = 128                    # channels per scale
E4M3_MAX = 448.0               # largest finite e4m3 value
TINY = 2.0 ** -126             # smallest scale: the smallest normal 32-bit number
EPS = 1e-6                     # the norm's epsilon
CLIP_EPS = 1e-6                # added to the gradient norm before the division
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def _functional():
    """The package's functional module (its folder is not an importable name, so it goes onto the path)."""
    folder = os.path.join(os.getcwd(), "deepsphere-weather_amd")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    from dsw_amd import functional

    return functional


# ---- cases ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the finest level of the U-Net (12 288 nodes, 8 samples) behind its first block, one training step of the norm
        {"name": "norm unet bf16", "kind": "norm", "rows": 98304, "channels": 256, "dtype": "bfloat16", "residual": True},
        # wide rows, generic: a long batch of tokens in training
        {"name": "norm wide bf16", "kind": "norm", "rows": 8192, "channels": 4096, "dtype": "bfloat16", "residual": True},
        # ragged small training batch in full precision, no residual in front
        {"name": "norm ragged fp32", "kind": "norm", "rows": 777, "channels": 1030, "dtype": "float32", "residual": False},
        # one token while serving: latency
        {"name": "norm8 one row", "kind": "norm_fp8", "rows": 1, "channels": 4096, "dtype": "bfloat16", "residual": True},
        # the finest level of the U-Net while serving
        {"name": "norm8 unet", "kind": "norm_fp8", "rows": 98304, "channels": 256, "dtype": "bfloat16", "residual": True},
        # one token through a square projection: bound by reading the weights
        {"name": "mix8 one row", "kind": "mix_fp8", "rows": 1, "k": 4096, "n": 4096, "dtype": "bfloat16", "bias": False},
        # a few requests decoded together
        {"name": "mix8 few rows", "kind": "mix_fp8", "rows": 48, "k": 4096, "n": 6144, "dtype": "bfloat16", "bias": False},
        # odd sizes in every direction, 32-bit output
        {"name": "mix8 ragged", "kind": "mix_fp8", "rows": 333, "k": 1100, "n": 1000, "dtype": "float32", "bias": True},
        # the residual branch of the U-Net's widest decoder block: its middle level at 8 samples, 512 -> 128 channels
        {"name": "mix8 unet", "kind": "mix_fp8", "rows": 24576, "k": 512, "n": 128, "dtype": "bfloat16", "bias": True},
        # a long prompt through a wide projection: bound by the matrix cores
        {"name": "mix8 large", "kind": "mix_fp8", "rows": 8192, "k": 4096, "n": 8192, "dtype": "bfloat16", "bias": False},
        # the U-Net's gradients, back to back in one flat buffer: latency
        {"name": "clip unet", "kind": "clip", "tensors": 44, "elements": 1770000, "dtype": "float32", "gap": 0, "norm": 5.0,
         "max_norm": 1.0, "p": 2.0},
        # many tensors of both types, each with an allocation of its own
        {"name": "clip many", "kind": "clip", "tensors": 320, "elements": 200000000, "dtype": "mixed", "gap": 64, "norm": 40.0,
         "max_norm": 1.0, "p": 2.0},
    ]


def _spread(rng, low, high):
    """A whole number spread evenly over the logarithm of [low, high]."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_fp8", "mix_fp8", "clip"])
    dtype = rng.choice(["float32", "bfloat16"])
    if kind in ("norm", "norm_fp8"):
        channels = _spread(rng, 16, 8192)
        rows = _spread(rng, 1, min(120000, (1 << 24) // channels))
        return {"kind": kind, "rows": rows, "channels": channels, "dtype": dtype, "residual": rng.random() < 0.7}
    if kind == "mix_fp8":
        k, n = _spread(rng, 16, 8192), _spread(rng, 16, 8192)
        rows = _spread(rng, 1, min(100000, (1 << 25) // n, (1 << 27) // k))
        return {"kind": kind, "rows": rows, "k": k, "n": n, "dtype": dtype, "bias": rng.random() < 0.5}
    tensors = _spread(rng, 1, 400)
    elements = tensors * _spread(rng, 8, 100000000 // tensors)
    return {"kind": kind, "tensors": tensors, "elements": elements, "dtype": rng.choice(["float32", "bfloat16", "mixed"]),
            "gap": rng.choice([0, 0, 3, 64]), "norm": rng.choice([0.5, 3.0, 20.0]), "max_norm": 1.0,
            "p": rng.choice([2.0, 2.0, math.inf, 1.0])}


def _blocks(channels):
    return -(-channels // BLOCK)


def _segments(case):
    """[(type's name, first element, elements)] of the gradients: log-normal sizes, each in the flat buffer of its type."""
    rng = random.Random(case["elements"] * 1009 + case["tensors"])
    weights = [math.exp(rng.gauss(0.0, 1.5)) for _ in range(case["tensors"])]
    total, end, made = sum(weights), {"float32": 0, "bfloat16": 0}, []
    for i, w in enumerate(weights):
        name = case["dtype"] if case["dtype"] != "mixed" else "float32" if i % 4 == 0 else "bfloat16"
        size = max(1, int(case["elements"] * w / total))
        if case["gap"] >= 64:                       # allocations of their own start on 256 bytes
            end[name] = -(-end[name] // 128) * 128
        made.append((name, end[name], size))
        end[name] += size + case["gap"]
    return made, end


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _normal(shape, gen, scale=1.0):
    return torch.randn(shape, generator=gen, device=DEV) * scale


def _activations(rows, channels, gen, dtype):
    """Activations as a network has them: normal, a few channels an order of magnitude larger."""
    x = _normal((rows, channels), gen)
    loud = torch.rand(channels, generator=gen, device=DEV) < 0.01
    return (x * torch.where(loud, 12.0, 1.0)).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    state = {"case": case}
    if kind in ("norm", "norm_fp8"):
        dtype, rows, channels = TYPES[case["dtype"]], case["rows"], case["channels"]
        state["x"] = _activations(rows, channels, gen, dtype)
        state["residual"] = _normal((rows, channels), gen, 3.0).to(dtype) if case["residual"] else None
        state["weight"] = (1.0 + _normal((channels,), gen, 0.2)).to(dtype)
        if kind == "norm":
            state["dy"] = _normal((rows, channels), gen, 0.1).to(dtype)
            state["dh"] = _normal((rows, channels), gen, 0.1).to(dtype) if case["residual"] else None
            for name in ("x", "residual", "weight"):
                if state[name] is not None:
                    state[name].requires_grad_()
    elif kind == "mix_fp8":
        rows, k, n = case["rows"], case["k"], case["n"]
        kb, nb = _blocks(k), _blocks(n)
        # activations and weights as they leave a quantiser: per block the largest value sits at 448
        x = torch.nn.functional.pad(_activations(rows, k, gen, torch.float32), (0, kb * BLOCK - k)).view(rows, kb, BLOCK)
        xs = (x.abs().amax(2) / E4M3_MAX).clamp_min(TINY)
        state["xq"] = (x / xs[..., None]).view(rows, kb * BLOCK)[:, :k].to(torch.float8_e4m3fn).contiguous()
        state["xs"] = xs.t().contiguous().t()                 # scales lie block after block, rows next to each other
        w = torch.nn.functional.pad(_normal((n, k), gen, k ** -0.5), (0, kb * BLOCK - k, 0, nb * BLOCK - n))
        w = w.view(nb, BLOCK, kb, BLOCK)
        ws = (w.abs().amax((1, 3)) / E4M3_MAX).clamp_min(TINY)
        state["wq"] = (w / ws[:, None, :, None]).view(nb * BLOCK, kb * BLOCK)[:n, :k].to(torch.float8_e4m3fn).contiguous()
        state["ws"] = ws.contiguous()
        state["bias"] = _normal((n,), gen).to(TYPES[case["dtype"]]) if case["bias"] else None
    else:
        made, end = _segments(case)
        flat = {name: torch.zeros(max(1, length), dtype=TYPES[name], device=DEV) for name, length in end.items()}
        loud = torch.exp(torch.randn(len(made), generator=torch.Generator().manual_seed(seed)) * 1.5).tolist()
        unit = math.sqrt(sum(a * a * size for a, (_, _, size) in zip(loud, made)))
        state["grads"] = [flat[name][first:first + size] for name, first, size in made]
        for g, a in zip(state["grads"], loud):
            g.copy_(_normal(g.shape, gen, case["norm"] * a / unit))
        state["flat"] = {name: torch.zeros_like(t) for name, t in flat.items() if end[name]}
        state["out"] = [state["flat"][name][first:first + size] for name, first, size in made]
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------------
def _plain_norm(s):
    x, r, w = s["x"].detach(), s["residual"], s["weight"].detach().float()
    h = x.float() if r is None else x.float() + r.detach().float()
    rstd = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    xhat = h * rstd
    gw = s["dy"].float() * w
    dx = rstd * (gw - xhat * (gw * xhat).mean(1, keepdim=True))
    dw = (s["dy"].float() * xhat).sum(0)
    out = {"y": (xhat * w).to(x.dtype), "dw": dw.to(x.dtype)}
    if r is None:
        return {**out, "dx": dx.to(x.dtype)}
    dx = (dx + s["dh"].float()).to(x.dtype)
    return {**out, "h": h.to(x.dtype), "dx": dx, "dresidual": dx}


def _own_norm(s):
    F = _functional()
    if s["residual"] is None:
        y = F.rms_norm(s["x"], s["weight"], EPS)
        dx, dw = torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw}
    y, h = F.rms_norm_residual(s["x"], s["residual"], s["weight"], EPS)
    dx, dr, dw = torch.autograd.grad((y, h), (s["x"], s["residual"], s["weight"]), (s["dy"], s["dh"]))
    return {"y": y, "h": h, "dx": dx, "dresidual": dr, "dw": dw}


def _plain_norm_fp8(s):
    x, r = s["x"], s["residual"]
    rows, channels = x.shape
    kb = _blocks(channels)
    h = x.float() if r is None else x.float() + r.float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["weight"].float()
    y = torch.nn.functional.pad(y, (0, kb * BLOCK - channels)).view(rows, kb, BLOCK)
    scale = (y.abs().amax(2) / E4M3_MAX).clamp_min(TINY)
    q = (y / scale[..., None]).view(rows, kb * BLOCK)[:, :channels].to(torch.float8_e4m3fn)
    return {"q": q, "scale": scale} if r is None else {"q": q, "scale": scale, "h": h.to(x.dtype)}


def _own_norm_fp8(s):
    rows, h = _functional().rms_norm_fp8(s["x"], s["weight"], residual=s["residual"], eps=EPS)
    return {"q": rows.q, "scale": rows.scale} if h is None else {"q": rows.q, "scale": rows.scale, "h": h}


def _plain_mix(s):
    k, n = s["wq"].shape[1], s["wq"].shape[0]
    x = s["xq"].float() * s["xs"].repeat_interleave(BLOCK, 1)[:, :k]
    w = s["wq"].float() * s["ws"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = x @ w.t()
    y = y if s["bias"] is None else y + s["bias"].float()
    return y.to(TYPES[s["case"]["dtype"]])


def _own_mix(s):
    F = _functional()
    return F.dense_mix_fp8(F.Fp8Rows(s["xq"], s["xs"]), F.Fp8Weight(s["wq"], s["ws"]), s["bias"], dtype=TYPES[s["case"]["dtype"]])


def _plain_clip(s):
    p = s["case"]["p"]
    if math.isinf(p):
        norm = torch.stack([g.abs().max() for g in s["grads"]]).double().max()
    elif p == 1.0:
        norm = torch.stack([g.double().abs().sum() for g in s["grads"]]).sum()
    else:
        norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt()
    scale = (s["case"]["max_norm"] / (norm + CLIP_EPS)).clamp_max(1.0).float()
    [o.copy_(g.float() * scale) for o, g in zip(s["out"], s["grads"])]
    return {"norm": norm.float(), **s["flat"]}


def _own_clip(s):
    norm = _functional().clip_grad_norm_(s["grads"], s["case"]["max_norm"], s["case"]["p"], out=s["out"])
    return {"norm": norm, **s["flat"]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"norm": _own_norm, "norm_fp8": _own_norm_fp8, "mix_fp8": _own_mix, "clip": _own_clip}[kind](state)
    return {"norm": _plain_norm, "norm_fp8": _plain_norm_fp8, "mix_fp8": _plain_mix, "clip": _plain_clip}[kind](state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    size = {"float32": 4, "bfloat16": 2}
    if kind == "norm":
        e = size[case["dtype"]]
        n = case["rows"] * case["channels"]
        # x, dy in, y, dx out; with a residual also r, dh in, h out; the weight and its gradient once
        return {"bytes": n * e * (7 if case["residual"] else 4) + 2 * case["channels"] * e, "flops": 14 * n}
    if kind == "norm_fp8":
        e = size[case["dtype"]]
        n = case["rows"] * case["channels"]
        return {"bytes": n * (e * (3 if case["residual"] else 1) + 1) + case["rows"] * _blocks(case["channels"]) * 4
                + case["channels"] * e, "flops": 8 * n}
    if kind == "mix_fp8":
        m, k, n, e = case["rows"], case["k"], case["n"], size[case["dtype"]]
        return {"bytes": m * k + n * k + m * n * e + 4 * _blocks(k) * (m + _blocks(n)) + (n * e if case["bias"] else 0),
                "flops": 2 * m * n * k}
    made, _ = _segments(case)
    return {"bytes": sum(2 * n * size[name] for name, _, n in made), "flops": 3 * sum(n for _, _, n in made)}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def _exact_norm(s):
    w = s["weight"].detach().double()
    h = s["x"].detach().double()
    if s["residual"] is not None:
        h = h + s["residual"].detach().double()
    c = h.shape[1]
    length = torch.sqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True).square() / c + EPS)
    unit = h / length
    g = s["dy"].double()
    along = torch.linalg.vecdot(g * w, unit).unsqueeze(1) / c
    dx = (g * w - along * unit) / length
    got = {"y": unit * w, "dw": torch.linalg.vecdot(g, unit, dim=0)}
    if s["residual"] is None:
        return {**got, "dx": dx}
    dx = dx + s["dh"].double()
    return {**got, "h": h, "dx": dx, "dresidual": dx}


def _exact_norm_fp8(s):
    h = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
    c = h.shape[1]
    y = h / torch.sqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True).square() / c + EPS) * s["weight"].double()
    scales = [torch.clamp(part.abs().max(dim=1).values / E4M3_MAX, min=TINY) for part in y.split(BLOCK, dim=1)]
    q = torch.cat([part / t[:, None] for part, t in zip(y.split(BLOCK, dim=1), scales)], dim=1)
    got = {"q": q, "scale": torch.stack(scales, dim=1)}       # q before its rounding to e4m3
    return got if s["residual"] is None else {**got, "h": h}


def _exact_mix(s):
    n, k = s["wq"].shape
    y = torch.zeros(s["xq"].shape[0], n, dtype=torch.float64, device=DEV)
    owner = torch.arange(n, device=DEV) // BLOCK
    for b in range(_blocks(k)):
        part = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
        w = s["wq"][:, part].double().t().contiguous()
        y += (s["xq"][:, part].double() @ w) * (s["xs"][:, b].double()[:, None] * s["ws"][:, b].double()[owner][None, :])
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_clip(s):
    p, total = s["case"]["p"], 0.0
    for g in s["grads"]:
        v = float(torch.linalg.vector_norm(g.double(), ord=p))
        total = max(total, v) if math.isinf(p) else total + v ** p
    norm = total if math.isinf(p) else total ** (1.0 / p)
    factor = min(1.0, s["case"]["max_norm"] / (norm + CLIP_EPS))
    wide = {name: torch.zeros(t.numel(), dtype=torch.float64, device=DEV) for name, t in s["flat"].items()}
    for (name, first, size), g in zip(_segments(s["case"])[0], s["grads"]):
        wide[name][first:first + size] = g.double() * factor
    return {"norm": torch.tensor(norm, dtype=torch.float64), **wide}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "norm_fp8": _exact_norm_fp8, "mix_fp8": _exact_mix, "clip": _exact_clip}[case["kind"]](s)

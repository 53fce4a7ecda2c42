"""Measured cases of the image and video block operators: group norm with an activation
over channels-last maps (and its gradient), the rotary rotation of queries and keys by
several position axes (and its gradient, the inverse rotation), and attention over all
tokens of a map.

`run` computes a case in its plain form (elementary torch operations in 32 bits, rounded
once at the end) or, with `own` set, through the package's operators. The channel widths
(64 to 512), the head width 32 and the 1920x1080 frames padded to 1920x1088 are the
network's own; the other sizes are generic.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
THETA = 100.0  # base of the position frequencies: periods from 2 pi to about 600 cells of a map


def listed():
    return [
        # group norm + SiLU of the deepest map of a small picture: one launch's latency
        {"name": "norm 8x8x512", "op": "norm", "n": 1, "l": 64, "c": 512, "groups": 32, "act": "silu", "dtype": "fp16"},
        # an odd map with ten channels a group (320 = 32 x 10), three pictures
        {"name": "norm 135x241x320", "op": "norm", "n": 3, "l": 135 * 241, "c": 320, "groups": 32, "act": "silu",
         "dtype": "bf16"},
        # the full-resolution map of two 1920x1080 frames, larger than any cache
        {"name": "norm 1088x1920x64", "op": "norm", "n": 2, "l": 1088 * 1920, "c": 64, "groups": 16, "act": "silu",
         "dtype": "fp16"},
        # gradients at a small odd crop, as in fine-tuning in 32 bits
        {"name": "norm grad 33x47x96", "op": "norm_grad", "n": 2, "l": 33 * 47, "c": 96, "groups": 8, "act": "gelu",
         "dtype": "fp32"},
        # gradients of the 1/8-resolution map of four frames
        {"name": "norm grad 136x240x512", "op": "norm_grad", "n": 4, "l": 136 * 240, "c": 512, "groups": 32,
         "act": "silu", "dtype": "fp16"},
        # one new token: latency
        {"name": "rotary one token", "op": "rotary", "b": 1, "l": 1, "h": 16, "hk": 16, "d": 64, "axes": 2, "rest": 0,
         "start": 57, "layout": "half", "packed": False, "inverse": False, "dtype": "bf16"},
        # the 1/8-resolution map of a frame, q and k inside one packed qkv, the network's 32-wide heads
        {"name": "rotary 136x240 packed", "op": "rotary", "b": 1, "l": 136 * 240, "h": 16, "hk": 16, "d": 32,
         "axes": 2, "rest": 0, "start": 0, "layout": "axial", "packed": True, "inverse": False, "dtype": "fp16"},
        # gradients of a clip's queries and (fewer) keys: time, height and width, an odd number of cells
        {"name": "rotary grad clip", "op": "rotary", "b": 2, "l": 9 * 45 * 79, "h": 12, "hk": 4, "d": 128, "axes": 3,
         "rest": 2, "start": 0, "layout": "interleaved", "packed": False, "inverse": True, "dtype": "bf16"},
        # the 1/32-resolution maps of four frames, 32-wide heads
        {"name": "attention 34x60", "op": "attention", "b": 4, "lq": 34 * 60, "lk": 34 * 60, "h": 16, "hk": 16,
         "d": 32, "masked": False, "packed": True, "dtype": "fp16"},
        # three pictures of different sizes in one batch, padded: masked keys, one picture absent
        {"name": "attention 39x39 masked", "op": "attention", "b": 3, "lq": 39 * 39, "lk": 39 * 39, "h": 12, "hk": 4,
         "d": 64, "masked": True, "packed": False, "dtype": "bf16"},
        # the 1/16-resolution map of a frame, wide heads: bound by the products
        {"name": "attention 68x120", "op": "attention", "b": 1, "lq": 68 * 120, "lk": 68 * 120, "h": 8, "hk": 8,
         "d": 128, "masked": False, "packed": True, "dtype": "bf16"},
        # one summary token a picture reads the 1/8-resolution map of a frame
        {"name": "attention one query", "op": "attention", "b": 2, "lq": 1, "lk": 136 * 240, "h": 16, "hk": 16,
         "d": 64, "masked": False, "packed": False, "dtype": "fp16"},
    ]


def _between(rng, lo, hi):
    """A whole number, spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "rotary", "rotary", "attention", "attention"])
    dtype = rng.choice(["fp16", "bf16", "fp32"])
    if op in ("norm", "norm_grad"):
        groups = rng.choice([1, 4, 8, 16, 32])
        c = groups * _between(rng, 2, 512 // groups)
        n = rng.randint(1, 5)
        most = (1 << 26) if op == "norm_grad" else (1 << 28)
        if dtype == "fp32":
            most //= 2
        return {"op": op, "n": n, "l": _between(rng, 1, min(1088 * 1920, most // (n * c))), "c": c, "groups": groups,
                "act": rng.choice(["none", "relu", "silu", "gelu"]), "dtype": dtype}
    if op == "rotary":
        axes = rng.randint(1, 3)
        d = 8 * rng.randint(1, 16)
        hk = rng.choice([1, 2, 4, 8, 16])
        packed = rng.random() < 0.4
        h = hk if packed else hk * rng.choice([1, 1, 2, 4])
        b = rng.randint(1, 4)
        return {"op": op, "b": b, "l": _between(rng, 1, min(100000, (1 << 26) // (b * (h + hk) * d))), "h": h, "hk": hk,
                "d": d, "axes": axes, "rest": rng.choice([0, 0, 1, 2]), "start": rng.randint(0, 64),
                "packed": packed,
                "layout": rng.choice(["half", "interleaved", "axial"]), "inverse": rng.random() < 0.4, "dtype": dtype}
    b = rng.randint(1, 4)
    hk = rng.choice([1, 2, 4, 8])
    h = hk * rng.choice([1, 1, 2, 3])
    most = (1 << 29) // (b * h)  # scores of a head: the plain form holds all of them
    lk = _between(rng, 1, 40000)
    lq = _between(rng, 1, max(1, min(8192, most // lk)))
    packed = lq > 64 and lk <= 8192 and lk * lk <= most and rng.random() < 0.5
    if packed:
        lq, h = lk, hk
    return {"op": op, "b": b, "lq": lq, "lk": lk, "h": h, "hk": hk, "d": rng.choice([16, 32, 40, 64, 80, 96, 128]),
            "masked": rng.random() < 0.4, "packed": packed, "dtype": "bf16" if dtype == "fp32" else dtype}


def _sections(case):
    """Pairs of channels that turn with each axis; `rest` pairs of a head do not turn."""
    pairs = max(case["axes"], case["d"] // 2 - case["rest"])
    each = pairs // case["axes"]
    return [pairs - each * (case["axes"] - 1)] + [each] * (case["axes"] - 1)


def _cells(case, dev):
    """Positions [l, axes] of the cells of a clip, time first; the last frame may be ragged."""
    side = max(1, min(240, int(math.ceil(case["l"] ** (1.0 / case["axes"])))))
    i = torch.arange(case["l"], device=dev)
    last = [i // side ** (case["axes"] - 1)] + [i // side ** (case["axes"] - 1 - a) % side
                                                for a in range(1, case["axes"])]
    return torch.stack(last, 1).to(torch.int32) + case["start"]


def _seen(case):
    """Of each picture of a padded batch: the batch's width, the picture's, and the tokens before its lower
    padding. Every further picture is a quarter smaller each way; the last of several is absent."""
    side, seen = max(1, math.isqrt(case["lk"])), []
    for i in range(case["b"]):
        share = 0.0 if 0 < i == case["b"] - 1 else 0.75 ** i
        seen.append((side, math.ceil(share * side), math.ceil(share * case["lk"])))
    return seen


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    s = {"case": case, "seed": seed}
    if case["op"] in ("norm", "norm_grad"):
        n, l, c, groups = case["n"], case["l"], case["c"], case["groups"]
        # activations: every channel with its own level and spread
        s["x"] = (normal(n, l, c) * (0.5 + normal(c).abs()) + normal(c)).to(dt)
        s["weight"] = 1 + 0.2 * normal(c)
        s["bias"] = 0.2 * normal(c)
        if case["op"] == "norm_grad":
            s["dy"] = normal(n, l, c).to(dt)
            # what the forward pass kept: mean and 1 / standard deviation of each picture's groups
            per = s["x"].view(n, l, groups, c // groups)
            mean = per.mean((1, 3), dtype=torch.float32)
            var = (per.float() - mean.view(n, 1, groups, 1)).square_().mean((1, 3))
            s["mean"], s["rstd"] = mean, (var + EPS).rsqrt()
    elif case["op"] == "rotary":
        b, l, h, hk, d = (case[k] for k in ("b", "l", "h", "hk", "d"))
        if case["packed"]:
            s["q"], s["k"], _ = normal(b, l, 3, h, d).to(dt).unbind(2)
        else:
            s["q"], s["k"] = normal(b, l, h, d).to(dt), normal(b, l, hk, d).to(dt)
        s["sections"] = _sections(case)
        s["positions"] = _cells(case, dev)
        s["inv_freq"] = torch.cat([THETA ** (-torch.arange(m, device=dev) / m) for m in s["sections"]]).float()
    else:
        b, lq, lk, h, hk, d = (case[k] for k in ("b", "lq", "lk", "h", "hk", "d"))
        if case["packed"]:
            s["q"], s["k"], s["v"] = normal(b, lq, 3, h, d).to(dt).unbind(2)
        else:
            s["q"] = normal(b, lq, h, d).to(dt)
            s["k"], s["v"] = normal(b, lk, hk, d).to(dt), normal(b, lk, hk, d).to(dt)
        s["key_mask"] = None
        if case["masked"]:
            i = torch.arange(lk, device=dev)
            s["key_mask"] = torch.stack([(i % side < wide) & (i < first) for side, wide, first in _seen(case)])
    return s


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return sig * (1 + z * (1 - sig))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _plain_norm(s):
    case, x = s["case"], s["x"]
    n, l, c, groups = case["n"], case["l"], case["c"], case["groups"]
    per = x.float().view(n, l, groups, c // groups)
    mean = per.mean((1, 3), keepdim=True)
    per = per - mean
    rstd = (per.square().mean((1, 3), keepdim=True) + EPS).rsqrt()
    z = (per * rstd).view(n, l, c) * s["weight"] + s["bias"]
    return _act(z, case["act"]).to(x.dtype)


def _plain_norm_grad(s):
    case, x = s["case"], s["x"]
    n, l, c, groups = case["n"], case["l"], case["c"], case["groups"]
    mean, rstd = s["mean"].view(n, 1, groups, 1), s["rstd"].view(n, 1, groups, 1)
    hat = ((x.float().view(n, l, groups, c // groups) - mean) * rstd).view(n, l, c)
    dz = s["dy"].float() * _act_slope(hat * s["weight"] + s["bias"], case["act"])
    dweight, dbias = (dz * hat).sum((0, 1)), dz.sum((0, 1))
    dhat = (dz * s["weight"]).view(n, l, groups, c // groups)
    hat = hat.view(n, l, groups, c // groups)
    dx = rstd * (dhat - dhat.mean((1, 3), keepdim=True) - hat * (dhat * hat).mean((1, 3), keepdim=True))
    return dx.view(n, l, c).to(x.dtype), dweight, dbias


def _pair_channels(sections, layout, dev):
    """The first and the second channel of each pair."""
    pairs = sum(sections)
    p = torch.arange(pairs, device=dev)
    if layout == "interleaved":
        return 2 * p, 2 * p + 1
    if layout == "half":
        return p, p + pairs
    width = torch.tensor(sections, device=dev).repeat_interleave(torch.tensor(sections, device=dev))
    start = torch.tensor([sum(sections[:a]) for a in range(len(sections))], device=dev).repeat_interleave(
        torch.tensor(sections, device=dev))
    return p + start, p + start + width


def _turn(x, lo, hi, cos, sin):
    y = x.float()
    a, b = y[..., lo], y[..., hi]
    y = y.clone()
    y[..., lo] = a * cos - b * sin
    y[..., hi] = a * sin + b * cos
    return y.to(x.dtype)


def _plain_rotary(s):
    case, dev = s["case"], s["q"].device
    sections = s["sections"]
    lo, hi = _pair_channels(sections, case["layout"], dev)
    axis = torch.arange(len(sections), device=dev).repeat_interleave(torch.tensor(sections, device=dev))
    angle = s["positions"].float()[:, axis] * s["inv_freq"]
    cos, sin = angle.cos()[None, :, None], angle.sin()[None, :, None]
    if case["inverse"]:
        sin = -sin
    return _turn(s["q"], lo, hi, cos, sin), _turn(s["k"], lo, hi, cos, sin)


def _plain_attention(s):
    case = s["case"]
    share = case["h"] // case["hk"]
    q = s["q"].float().transpose(1, 2)
    k = s["k"].float().transpose(1, 2).repeat_interleave(share, 1)
    v = s["v"].float().transpose(1, 2).repeat_interleave(share, 1)
    scores = q @ k.transpose(2, 3) * case["d"] ** -0.5
    if s["key_mask"] is None:
        p = torch.exp(scores - scores.amax(3, keepdim=True))
        out = (p @ v) / p.sum(3, keepdim=True)
    else:
        seen = s["key_mask"][:, None, None, :]
        scores = torch.where(seen, scores, -torch.inf)
        top = scores.amax(3, keepdim=True)
        p = torch.exp(scores - torch.where(top == -torch.inf, 0.0, top))
        total = p.sum(3, keepdim=True)
        v = torch.where(s["key_mask"][:, None, :, None], v, 0.0)
        out = torch.where(total > 0, (p @ v) / total, 0.0)
    return out.transpose(1, 2).to(s["q"].dtype).contiguous()


_package = None


def _ops():
    global _package
    if _package is None:
        import importlib
        _package = importlib.import_module("scunet-rs_b200")
    return _package.ops


def run(s):
    case = s["case"]
    if not own:
        return {"norm": _plain_norm, "norm_grad": _plain_norm_grad, "rotary": _plain_rotary,
                "attention": _plain_attention}[case["op"]](s)
    ops = _ops()
    if case["op"] == "norm":
        return ops.group_norm(s["x"], case["groups"], s["weight"], s["bias"], eps=EPS, act=case["act"])
    if case["op"] == "norm_grad":
        return ops.group_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], case["groups"], s["weight"], s["bias"],
                                       act=case["act"])
    if case["op"] == "rotary":
        return ops.rotate_axes(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"], layout=case["layout"],
                               inverse=case["inverse"])
    return ops.attention(s["q"], s["k"], s["v"], key_mask=s["key_mask"])


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        values = case["n"] * case["l"] * case["c"]
        return {"bytes": 2 * values * size + 8 * case["c"], "flops": 14 * values}
    if case["op"] == "norm_grad":
        values = case["n"] * case["l"] * case["c"]
        return {"bytes": 3 * values * size + 16 * case["c"] + 8 * case["n"] * case["groups"], "flops": 28 * values}
    if case["op"] == "rotary":
        values = case["b"] * case["l"] * (case["h"] + case["hk"]) * case["d"]
        return {"bytes": 2 * values * size + 4 * case["l"] * case["axes"], "flops": 3 * values}
    b, lq, lk, h, hk, d = (case[k] for k in ("b", "lq", "lk", "h", "hk", "d"))
    keys = b * lk  # visible keys of all pictures
    if case["masked"]:
        keys = sum(first // side * wide + min(first % side, wide) for side, wide, first in _seen(case))
    return {"bytes": 2 * d * (2 * b * lq * h + 2 * keys * hk) + (b * lk if case["masked"] else 0),
            "flops": 4 * h * lq * keys * d}


def exact(case, seed):
    """The operators' definitions in 64 bits: the norm by its variance and its gradient by
    differentiation, the rotation as a product of complex numbers, attention head by head."""
    s = prepare(case, seed)
    if case["op"] in ("norm", "norm_grad"):
        n, l, c, groups = case["n"], case["l"], case["c"], case["groups"]
        grad = case["op"] == "norm_grad"
        outs, dw, db = [], 0.0, 0.0
        for k in range(n):  # one picture at a time bounds the memory
            x = s["x"][k].double().requires_grad_(grad)
            w, bias = s["weight"].double().requires_grad_(grad), s["bias"].double().requires_grad_(grad)
            per = x.reshape(l, groups, c // groups).transpose(0, 1).reshape(groups, -1)
            var, mean = torch.var_mean(per, 1, correction=0, keepdim=True)
            hat = ((per - mean) / torch.sqrt(var + EPS)).reshape(groups, l, c // groups).transpose(0, 1).reshape(l, c)
            z = hat * w + bias
            if case["act"] == "relu":
                y = torch.relu(z)
            elif case["act"] == "silu":
                y = z * torch.sigmoid(z)
            elif case["act"] == "gelu":
                y = z * torch.special.ndtr(z)
            else:
                y = z
            if grad:
                dx, a, b = torch.autograd.grad(y, (x, w, bias), s["dy"][k].double())
                outs.append(dx)
                dw, db = dw + a, db + b
            else:
                outs.append(y)
        return (torch.stack(outs), dw, db) if grad else torch.stack(outs)
    if case["op"] == "rotary":
        angles, at = [], 0
        for a, m in enumerate(s["sections"]):
            angles.append(s["positions"][:, a, None].double() * s["inv_freq"][at:at + m].double())
            at += m
        angle = torch.cat(angles, 1) * (-1 if case["inverse"] else 1)
        turn = torch.polar(torch.ones_like(angle), angle)[None, :, None]
        outs = []
        for x in (s["q"], s["k"]):
            x = x.double()
            y = x.clone()
            if case["layout"] == "interleaved":
                y[..., :2 * at] = torch.view_as_real(
                    torch.view_as_complex(x[..., :2 * at].reshape(*x.shape[:3], at, 2).contiguous()) * turn).flatten(3)
            elif case["layout"] == "half":
                z = torch.complex(x[..., :at], x[..., at:2 * at]) * turn
                y[..., :at], y[..., at:2 * at] = z.real, z.imag
            else:
                first = 0
                for m in s["sections"]:
                    z = torch.complex(x[..., 2 * first:2 * first + m], x[..., 2 * first + m:2 * first + 2 * m])
                    z = z * turn[..., first:first + m]
                    y[..., 2 * first:2 * first + m], y[..., 2 * first + m:2 * first + 2 * m] = z.real, z.imag
                    first += m
            outs.append(y)
        return tuple(outs)
    share = case["h"] // case["hk"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b in range(case["b"]):
        keep = slice(None) if s["key_mask"] is None else s["key_mask"][b].nonzero()[:, 0]
        for h in range(case["h"]):
            k, v = s["k"][b, :, h // share][keep].double(), s["v"][b, :, h // share][keep].double()
            if k.shape[0]:
                out[b, :, h] = torch.softmax(s["q"][b, :, h].double() @ k.t() / math.sqrt(case["d"]), 1) @ v
    return out

"""The channel operators' measured cases: ``blockcopy.linear_act`` (matrix product with bias, activation and residual in its epilogue) and
``blockcopy.norm_residual`` (the norms after one block and before the next, with the block's gate and the residual scale), forward and
backward.

``own`` false: the operators' plain forms, elementary torch operations in 32 bits rounded once at the end.  ``own`` true: the calls a user
makes of the package.  A row is one pixel of a channels-last map or one token; its features are the map's channels."""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "blockcopy-video-processing-pytorch_amd")
_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases
def _linear(name, dtype, m, k, n, act, bias=True, residual=False, train=False):
    return {"name": name, "op": "linear", "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "bias": bias, "residual": residual, "train": train}


def _norm(name, dtype, m, c, out_norm, in_norm, gate, scale=1.0, bias=False, groups=1, train=False, block=True):
    return {"name": name, "op": "norm", "dtype": dtype, "m": m, "c": c, "out_norm": out_norm, "in_norm": in_norm, "gate": gate, "groups": groups,
            "scale": scale, "bias": bias, "train": train, "block": block}


def listed():
    return [
        # one token (or the pooled vector of a frame) through a projection: latency and the weight's bytes
        _linear("linear bf16 1 row", "bf16", 1, 4096, 4096, "silu"),
        # a handful of regions through a classifier of an odd number of classes and features
        _linear("linear f16 13 rows odd", "f16", 13, 2047, 1001, "none"),
        # the skipped-tile remainder of a frame: 68 tiles of 16 x 16 pixels, 512 channels widened fourfold
        _linear("linear bf16 68 tiles", "bf16", 17408, 512, 2048, "gelu"),
        # the same tiles narrowed again, with the block's residual, at full precision
        _linear("linear f32 tiles residual", "f32", 17408, 768, 256, "none", residual=True),
        # a long batch of tokens through a wide projection
        _linear("linear bf16 long", "bf16", 16384, 4096, 8192, "gelu_tanh"),
        # training: a few maps' pixels, odd in every size, with residual
        _linear("linear f32 train odd", "f32", 4099, 515, 1001, "gelu", residual=True, train=True),
        # training: many pixels, few channels (the weight gradient's sum runs over 131072 rows)
        _linear("linear f16 train pixels", "f16", 131072, 256, 512, "gelu", residual=True, train=True),
        # training: a wide projection
        _linear("linear bf16 train wide", "bf16", 8192, 2048, 8192, "silu", train=True),
        # one token between two blocks
        _norm("norm bf16 1 row", "bf16", 1, 4096, "rms", "rms", "channel"),
        # executed tiles of a frame between two blocks: 68 tiles of 32 x 32 pixels, layer scale and LayerNorm before the next block
        _norm("norm f16 68 tiles", "f16", 69632, 256, "none", "layer", "channel", bias=True),
        # training: token rows of an odd width at full precision, a gate per sample
        _norm("norm f32 train odd", "f32", 5005, 1001, "layer", "rms", "sample", scale=0.7, bias=True, groups=7, train=True),
        # training: the residual stream of a long batch, a norm on both sides of the gate
        _norm("norm bf16 train long", "bf16", 32768, 2048, "rms", "rms", "channel", scale=1.0, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """A size spread over the logarithm of its range: odd as drawn, or brought to a multiple of 64 (channel counts mostly are one)."""
    v = _log_int(rng, lo, hi)
    if rng.random() < 0.5 and v >= 64:
        v = v // 64 * 64
    return v


def draw(rng):
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    train = rng.random() < 0.5
    if rng.random() < 0.5:
        m, k, n = _size(rng, 1, 131072), _size(rng, 16, 8192), _size(rng, 16, 8192)
        top = 1 << (33 if dtype == "f32" else 36)
        while m * k * n > top:
            m = max(1, m // 2)
        # (no gradient of relu: a pre-activation that is zero but for its rounding has either derivative)
        return {"op": "linear", "dtype": dtype, "m": m, "k": k, "n": n, "act": rng.choice(["none", "gelu", "gelu_tanh", "silu"] + ([] if train else ["relu"])),
                "bias": rng.random() < 0.8, "residual": rng.random() < 0.5, "train": train}
    m, c = _size(rng, 1, 131072), _size(rng, 16, 16384)
    while m * c > 1 << 26:
        m = max(1, m // 2)
    block = rng.random() < 0.85
    out_norm = rng.choice(["none", "rms", "layer"]) if block else "none"
    in_norm = rng.choice(["none", "rms", "layer"]) if block else rng.choice(["rms", "layer"])
    gate = rng.choice(["none", "channel", "sample"]) if block else "none"
    groups = 1
    if gate == "sample":
        groups = rng.choice([1, 2, 3, 5, 8])
        m = max(1, m // groups) * groups
    return {"op": "norm", "dtype": dtype, "m": m, "c": c, "out_norm": out_norm, "in_norm": in_norm, "gate": gate, "groups": groups,
            "scale": rng.choice([1.0, 0.7]) if block else 1.0, "bias": rng.random() < 0.5, "train": train, "block": block}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed) * 7919 + 11)
    dt = _DTYPES[case["dtype"]]

    def rand(*shape, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=g, device=dev) * std + mean).to(dt)

    st = {"case": dict(case)}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        st["x"] = rand(m, k)
        st["w"] = rand(n, k, std=k ** -0.5)
        st["b"] = rand(n, std=0.2) if case["bias"] else None
        st["r"] = rand(m, n) if case["residual"] else None
        st["gy"] = rand(m, n) if case["train"] else None
        leaves = ("x", "w", "b", "r")
    else:
        m, c = case["m"], case["c"]
        # the residual stream has a few channels that are far larger than the rest
        h = torch.randn((m, c), generator=g, device=dev)
        h[:, ::max(2, c // 3)] *= 8.0
        st["h"] = h.to(dt)
        st["y"] = rand(m, c, std=0.5, mean=0.1) if case["block"] else None
        st["wo"] = rand(c, std=0.2, mean=1.0) if case["out_norm"] != "none" else None
        st["bo"] = rand(c, std=0.1) if case["out_norm"] != "none" and case["bias"] else None
        st["wi"] = rand(c, std=0.2, mean=1.0) if case["in_norm"] != "none" else None
        st["bi"] = rand(c, std=0.1) if case["in_norm"] != "none" and case["bias"] else None
        st["gate"] = {"none": lambda: None, "channel": lambda: rand(c, std=0.3, mean=0.5),
                      "sample": lambda: rand(case["groups"], 1, c, std=0.3, mean=0.5)}[case["gate"]]()
        if case["gate"] == "sample":
            st["h"] = st["h"].view(case["groups"], m // case["groups"], c)
            st["y"] = st["y"].view(case["groups"], m // case["groups"], c)
        st["gh"] = rand(*st["h"].shape) if case["train"] and case["block"] else None
        st["gu"] = rand(*st["h"].shape) if case["train"] and case["in_norm"] != "none" else None
        leaves = ("h", "y", "wo", "bo", "gate", "wi", "bi")
    st["leaves"] = leaves
    if case["train"]:
        for name in leaves:
            if st[name] is not None:
                st[name].requires_grad_(True)
    return st


# ------------------------------------------------------------------------------------------------ the package's calls
def _run_own(st):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import blockcopy

    case = st["case"]
    leaves = [st[n] for n in st["leaves"] if st[n] is not None]
    with torch.set_grad_enabled(case["train"]):
        if case["op"] == "linear":
            y = blockcopy.linear_act(st["x"], st["w"], st["b"], activation=case["act"], residual=st["r"])
            if not case["train"]:
                return [y]
            return [y.detach(), *torch.autograd.grad(y, leaves, st["gy"])]
        h, u = blockcopy.norm_residual(st["h"], st["y"], out_norm=case["out_norm"], out_weight=st["wo"], out_bias=st["bo"], gate=st["gate"],
                                       residual_scale=case["scale"], in_norm=case["in_norm"], in_weight=st["wi"], in_bias=st["bi"], eps=_EPS)
        outs = ([h] if case["block"] else []) + ([u] if u is not None else [])
        if not case["train"]:
            return outs
        grads = torch.autograd.grad(outs, leaves, [t for t in (st["gh"], st["gu"]) if t is not None])
        return [*(o.detach() for o in outs), *grads]


# ------------------------------------------------------------------------------------------------ the plain forms
def _act(z, name):
    """Activation and its derivative."""
    if name == "none":
        return z, None
    if name == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if name == "gelu":
        phi = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        a = (2 / math.pi) ** 0.5
        t = torch.tanh(a * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)
    s = 1 / (1 + torch.exp(-z))
    return z * s, s * (1 + z * (1 - s))


def _plain_linear(st):
    case = st["case"]
    dt = st["x"].dtype
    x, w = st["x"].float(), st["w"].float()
    z = x @ w.t()
    if st["b"] is not None:
        z = z + st["b"].float()
    y, d = _act(z, case["act"])
    if st["r"] is not None:
        y = y + st["r"].float()
    out = [y.to(dt)]
    if case["train"]:
        gy = st["gy"].float()
        dz = gy if d is None else gy * d
        out += [(dz @ w).to(dt), (dz.t() @ x).to(dt)]
        if st["b"] is not None:
            out.append(dz.sum(0).to(dt))
        if st["r"] is not None:
            out.append(st["gy"])
    return out


def _plain_norm_fwd(x, kind, w, b):
    """Normalised rows, reciprocal deviation, and the norm's output."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)
    n = x * r
    o = n if w is None else n * w
    return n, r, o if b is None else o + b


def _plain_norm_bwd(g, n, r, kind):
    d = g - n * (g * n).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - g.mean(-1, keepdim=True)
    return d * r


def _plain_norm(st):
    case = st["case"]
    dt = st["h"].dtype
    f = {k: None if st[k] is None else st[k].float() for k in ("h", "y", "wo", "bo", "gate", "wi", "bi", "gh", "gu")}
    rows = tuple(range(f["h"].dim() - 1))
    h = f["h"]
    if case["block"]:
        t = f["y"]
        if case["out_norm"] != "none":
            ny, ry, t = _plain_norm_fwd(t, case["out_norm"], f["wo"], f["bo"])
        h = case["scale"] * h + (t if f["gate"] is None else f["gate"] * t)
    out = [h] if case["block"] else []
    if case["in_norm"] != "none":
        nh, rh, u = _plain_norm_fwd(h, case["in_norm"], f["wi"], f["bi"])
        out.append(u)
    if case["train"]:
        grads = {}
        g = f["gh"] if case["block"] else 0
        if case["in_norm"] != "none":
            grads["wi"], grads["bi"] = (f["gu"] * nh).sum(rows), f["gu"].sum(rows)
            g = g + _plain_norm_bwd(f["gu"] * f["wi"], nh, rh, case["in_norm"])
        grads["h"] = case["scale"] * g
        if case["block"]:
            dt_ = g
            if f["gate"] is not None:
                grads["gate"] = (g * t).sum(rows) if case["gate"] == "channel" else (g * t).sum(1, keepdim=True)
                dt_ = g * f["gate"]
            if case["out_norm"] != "none":
                grads["wo"], grads["bo"] = (dt_ * ny).sum(rows), dt_.sum(rows)
                dt_ = _plain_norm_bwd(dt_ * f["wo"], ny, ry, case["out_norm"])
            grads["y"] = dt_
        out += [grads[n] for n in st["leaves"] if st[n] is not None]
    return [o.to(dt) for o in out]


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_linear(state) if state["case"]["op"] == "linear" else _plain_norm(state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        mats = m * k + n * k + m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)
        if case["train"]:
            mats += m * n + m * k + n * k + (n if case["bias"] else 0)
        return {"bytes": e * mats, "flops": 2 * m * k * n * (3 if case["train"] else 1)}
    mc = case["m"] * case["c"]
    fwd = (3 if case["block"] else 1) + (1 if case["in_norm"] != "none" else 0)                   # h, y, new h; the next block's input
    bwd = ((3 if case["block"] else 1) + (1 if case["in_norm"] != "none" else 0)) if case["train"] else 0  # their gradients
    vec = case["c"] * sum([case["out_norm"] != "none", case["in_norm"] != "none", case["gate"] != "none"])
    return {"bytes": e * ((fwd + bwd) * mc + vec * (2 if case["train"] else 1)), "flops": mc * (12 + (24 if case["train"] else 0))}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    d = {k: v.detach().double().requires_grad_(case["train"]) for k, v in st.items() if isinstance(v, torch.Tensor)}
    get = d.get

    def normed(x, kind, w, b):
        if kind == "none":
            return x
        if kind == "layer":
            x = x - x.sum(-1, keepdim=True) / x.shape[-1]
        x = x * ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + _EPS) ** -0.5
        return (x if w is None else x * w) + (0 if b is None else b)

    with torch.set_grad_enabled(case["train"]):
        if case["op"] == "linear":
            z = torch.matmul(d["x"], d["w"].t()) + (0 if get("b") is None else d["b"])
            y = {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)),
                 "gelu": lambda: z * (torch.erf(z / math.sqrt(2)) + 1) / 2,
                 "gelu_tanh": lambda: z / 2 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))),
                 "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()
            outs, gs = [y + (0 if get("r") is None else d["r"])], [get("gy")]
        else:
            h = d["h"]
            if case["block"]:
                t = normed(d["y"], case["out_norm"], get("wo"), get("bo"))
                h = h * case["scale"] + (t if get("gate") is None else t * d["gate"])
            outs, gs = ([h], [get("gh")]) if case["block"] else ([], [])
            if case["in_norm"] != "none":
                outs, gs = outs + [normed(h, case["in_norm"], get("wi"), get("bi"))], gs + [get("gu")]
        if not case["train"]:
            return outs
        grads = torch.autograd.grad(outs, [d[n] for n in st["leaves"] if st[n] is not None], [g.detach() for g in gs])
    return [*(o.detach() for o in outs), *grads]

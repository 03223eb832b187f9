"""64-bit definitions of the channel operators with their gradients, and what rounding alone may put between them and a kernel.

U = 2^-24 is half a step of float32.  A sum of n terms in float32, in any order, is off by at most n U times the sum of the terms' sizes (first
order), and a value rounded to a type is off by eps / 2 of its size; every bound below adds up exactly such contributions."""
import math

import torch

U = 2.0 ** -24
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")
# largest size of the second derivative: gelu 2 phi(0) = 0.798, gelu_tanh just above it, silu 0.5; relu jumps only where z = 0 (exactly representable)
CURVE = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "gelu_tanh": 0.81, "silu": 0.5}


def half_eps(dtype):
    return torch.finfo(dtype).eps / 2


def rounded(v, err, dtype):
    """Bound of a value with error ``err`` after rounding to ``dtype``: half a step of its size, and never less than half the spacing of the
    type's numbers next to zero (its subnormal numbers lie smallest_normal * eps apart: float16 2^-24, half of it 2^-25)."""
    return err + half_eps(dtype) * (v.abs() + err) + half_eps(dtype) * torch.finfo(dtype).smallest_normal


def act(z, name):
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if name == "gelu":
        p = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * p, p + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        a, b = math.sqrt(2 / math.pi), 0.044715
        s = torch.sigmoid(2 * a * (z + b * z ** 3))
        return z * s, s + z * s * (1 - s) * 2 * a * (1 + 3 * b * z * z)
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s))


def linear(x, w, b, r, name, gy=None):
    """{name: (value, bound)} of y and, with gy, of dx, dw, db for inputs of one type (bias of its own)."""
    he, dtype = half_eps(x.dtype), x.dtype
    x, w = x.double(), w.double()
    K, N, M = w.shape[1], w.shape[0], x.shape[0]
    z = x @ w.t()
    size = x.abs() @ w.abs().t()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    dz_err = (K + 1) * U * size
    a, d = act(z, name)
    # an activation's own evaluation: at most 16 float32 roundings of numbers no larger than |z| + 1 times the result's scale
    y_err = 1.13 * dz_err + 16 * U * (z.abs() + a.abs())
    y = a
    if r is not None:
        y = y + r.double()
        y_err = y_err + U * (a.abs() + r.double().abs())
    out = {"y": (y, rounded(y, y_err, dtype))}
    if gy is not None:
        g = gy.double()
        # the derivative is taken at z rounded to the type; its own evaluation is off by at most 32 U (values up to 1.13, products of |z| e^-z2)
        e = g.abs() * (CURVE[name] * (dz_err + he * z.abs()) + (0.0 if name in ("none", "relu") else 32 * U))
        dz = g * d
        out["db"] = (dz.sum(0), e.sum(0) + (M + 1) * U * (dz.abs() + e).sum(0))
        if name != "none":
            e = rounded(dz, e, dtype)       # dz is stored in the type
        dx, dw = dz @ w, dz.t() @ x
        out["dx"] = (dx, e @ w.abs() + N * U * ((dz.abs() + e) @ w.abs()))
        out["dw"] = (dw, e.t() @ x.abs() + M * U * ((dz.abs() + e).t() @ x.abs()))
        for k, t in (("dx", dtype), ("dw", dtype), ("db", b.dtype if b is not None else dtype)):
            v, err = out[k]
            out[k] = (v, rounded(v, err, t))
    return out


def linear_gradients(x, w, b, name, gy):
    """{name: (value, bound)} of dx, dw, db where nothing but the result is rounded to the tensors' type: z in float32, dz = dy act'(z) as two numbers
    of the type (the second holds what the first leaves: off by half_eps^2 of dz)."""
    he, dtype = half_eps(x.dtype), x.dtype
    x, w, g = x.double(), w.double(), gy.double()
    K, N, M = w.shape[1], w.shape[0], x.shape[0]
    z = x @ w.t() + b.double()
    z_err = (K + 2) * U * (x.abs() @ w.abs().t() + b.double().abs())
    d = act(z, name)[1]
    # (the derivative's own evaluation: at most 32 U, as in linear())
    e = g.abs() * (CURVE[name] * z_err + 32 * U)
    dz = g * d
    out = {"db": (dz.sum(0), e.sum(0) + (M + 1) * U * (dz.abs() + e).sum(0))}
    e = e + he * he * (dz.abs() + e) + 2.0 ** -34 * he
    out["dx"] = (dz @ w, e @ w.abs() + 2 * N * U * ((dz.abs() + e) @ w.abs()))
    out["dw"] = (dz.t() @ x, e.t() @ x.abs() + 2 * M * U * ((dz.abs() + e).t() @ x.abs()))
    return {k: (v, rounded(v, err, b.dtype if k == "db" else dtype)) for k, (v, err) in out.items()}


def normed(x, kind, w, b, eps):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    x = x if w is None else x * w
    return x if b is None else x + b


def norm_residual(h, y, p, gate, scale, out_norm, in_norm, eps, rows_per_gate=0):
    """(h', u) in 64 bits out of 64-bit tensors (rows, C); p = {"wo", "bo", "wi", "bi"}; gate (C,) or (groups, C)."""
    if y is not None:
        t = normed(y, out_norm, p.get("wo"), p.get("bo"), eps)
        if gate is not None:
            g = gate if not rows_per_gate else gate.repeat_interleave(rows_per_gate, 0)
            t = t * g
        h = scale * h + t
    u = None if in_norm == "none" else normed(h, in_norm, p.get("wi"), p.get("bi"), eps)
    return h, u

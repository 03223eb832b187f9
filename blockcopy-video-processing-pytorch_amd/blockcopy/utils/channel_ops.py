"""Channel operators: what a residual network of row products is made of, on plain tensors and on packed tiles (NOT part of the reference's
API: an addition).

``linear_act``      y = act(x W^T + b) + residual: a 1x1 conv / linear layer with its whole epilogue in the product's kernel.
``norm_residual``   h' = residual_scale * h + gate * N_out(y),  u = N_in(h'): the norm after one block, the block's gate, the residual
                    stream and the norm before the next block in one pass.

Both work on rows of features: the last axis of a tensor (``dim=-1``, tokens), or axis 1 of a (N, C, H, W) map (``dim=1``, pixels), for which
channels-last memory is the free layout.  A packed or dense ``TensorWrapper`` is always read along axis 1 and gives a ``TensorWrapper``: rows
are independent of each other, so no halo, no transfer and no cache is involved, and skipped tiles keep their values when the result is
combined (in a frame sized for a ceiling of tiles every row is computed, the surplus ones out of whatever they hold).  float32, float16 and
bfloat16; sums, statistics, activations and everything between input and output in float32.  GPU tensors only.

Both are differentiable once with respect to every tensor argument.  Gradients of a captured graph follow torch's rule for captured
backward passes: warm up on the capturing stream, with no eager graph over the same leaves alive.  No call waits for the device, and every
result is run-to-run identical (sums are split and joined in a fixed order, no atomics)."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from blockcopy.backend import BlockCopyBackendError, get_backend
from blockcopy.core.tensorwrapper import TensorWrapper

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
NORMS = {"none": 0, "rms": 1, "layer": 2}
MAX_NORM_CHANNELS = 16384
_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def _backend(x):
    be = get_backend()
    if not x.is_cuda and be.name == "hip":
        raise BlockCopyBackendError("channel operators need GPU tensors (no CPU path)")
    return be


def _plain(t):
    """Plain-tensor view of an argument; pending work of a TensorWrapper is executed first."""
    if t is None or type(t) is torch.Tensor or type(t) is torch.nn.Parameter:
        return t
    if hasattr(t, "_plain"):
        return t._plain()
    return t.as_subclass(torch.Tensor) if isinstance(t, torch.Tensor) else t


def _features(x, dim, name):
    """x with its features last."""
    if dim == -1 or dim == x.dim() - 1:
        if x.dim() < 1:
            raise ValueError(f"{name}: a tensor with a feature axis is needed, got a scalar")
        return x
    if dim == 1 and x.dim() == 4:
        return x.permute(0, 2, 3, 1)
    raise ValueError(f"{name}: features are the last axis (dim=-1) or axis 1 of a (N, C, H, W) map (dim=1), got dim={dim} for shape {tuple(x.shape)}")


def _rows(x):
    """(rows, features) view of x, or of a contiguous copy where its strides allow none (features apart, overlapping rows)."""
    f = x.shape[-1]
    if x.dim() == 2 and x.is_contiguous():
        return x
    if x.dim() != 2:
        try:
            x = x.view(-1, f) if x.numel() else x.reshape(x.numel() // f if f else 0, f)
        except RuntimeError:
            x = x.reshape(-1, f)
    if (f > 1 and x.stride(1) != 1) or (x.shape[0] > 1 and x.stride(0) < f):
        x = x.contiguous()
    return x


def _matching(name, t, shape, like, what):
    if not isinstance(t, torch.Tensor) or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: {what} must have the shape {tuple(shape)} (features last; nothing is broadcast), got "
                         f"{tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__}")
    if t.dtype != like.dtype or t.device != like.device:
        raise TypeError(f"{name}: {what} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")


def _vector(name, p, n, like, what):
    """Per-channel parameter: n elements, the rows' dtype or float32."""
    if p is None:
        return None
    p = _plain(p)
    if not isinstance(p, torch.Tensor) or tuple(p.shape) != (n,):
        raise ValueError(f"{name}: {what} must be a vector of {n} channels, got {tuple(p.shape) if isinstance(p, torch.Tensor) else p!r}")
    if p.dtype not in (like.dtype, torch.float32) or p.device != like.device:
        raise TypeError(f"{name}: {what} must be {like.dtype} or float32 on {like.device}, got {p.dtype} on {p.device}")
    return p.contiguous()


def _wrapped(like, out, dim):
    """Rows (features last) back into the argument's axis order and kind."""
    if out is None:
        return None
    if dim == 1:
        out = out.permute(0, 3, 1, 2)
    if like is not None:
        return TensorWrapper._wrap_like(out, like, like.is_blocks)
    return out


def _argument(x, dim, name):
    """(plain tensor with features last, TensorWrapper or None, effective dim)"""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name}: a tensor is needed, got {type(x).__name__}")
    wrapper = x if isinstance(x, TensorWrapper) and x.is_init else None
    if wrapper is not None:
        dim = 1
    x = _plain(x)
    if x.dtype not in _DTYPES:
        raise TypeError(f"{name}: float32, float16 or bfloat16 tensors, got {x.dtype}")
    f = _features(x, dim, name)
    if dim == x.dim() - 1:
        dim = -1
    if f.shape[-1] == 0:
        raise ValueError(f"{name}: no features in shape {tuple(x.shape)}")
    return f, wrapper, dim


# ------------------------------------------------------------------------------------------------ product
class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, be):
        keep = act != 0 and any(ctx.needs_input_grad[:3])
        y, z = be.linear_fwd(x, weight, bias, act, residual, keep)
        ctx.save_for_backward(x if ctx.needs_input_grad[1] else None, weight if ctx.needs_input_grad[0] else None, z)
        ctx.act, ctx.be, ctx.shape = act, be, (x.shape[0], weight.shape[0], weight.shape[1])
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, weight, z = ctx.saved_tensors
        want = ctx.needs_input_grad
        dx = dw = db = None
        if any(want[:3]):
            dx, dw, db = ctx.be.linear_bwd(_rows(gy), z, x, weight, ctx.act, want[:3], ctx.bias_dtype)
        return dx, dw, db, gy if want[3] else None, None, None


def linear_act(x, weight, bias=None, activation: str = "none", residual=None, dim: int = -1):
    """``act(x W^T + bias) + residual`` over the features of ``x``.

    weight (out, in), or (out, in, 1, 1) as a 1x1 conv keeps it, in x's dtype; bias (out,) in x's dtype or float32; activation one of
    ``none relu gelu gelu_tanh silu``; residual of the result's shape.  Any number of rows (none among them), any sizes, row strides as they
    come.  Under autograd the pre-activations are kept in x's dtype for the backward pass."""
    name = "linear_act"
    if activation not in ACTIVATIONS:
        raise ValueError(f"{name}: activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    xf, wrapper, dim = _argument(x, dim, name)
    weight = _plain(weight)
    if weight.dim() == 4 and tuple(weight.shape[2:]) == (1, 1):
        weight = weight.flatten(1)
    if weight.dim() != 2 or weight.shape[1] != xf.shape[-1] or weight.shape[0] == 0:
        raise ValueError(f"{name}: weight must be (out, {xf.shape[-1]}), got {tuple(weight.shape)}")
    if weight.dtype != xf.dtype or weight.device != xf.device:
        raise TypeError(f"{name}: weight must be {xf.dtype} on {xf.device}, got {weight.dtype} on {weight.device}")
    bias = _vector(name, bias, weight.shape[0], xf, "bias")
    shape = (*xf.shape[:-1], weight.shape[0])
    res = None
    if residual is not None:
        res = _features(_plain(residual), dim, name)
        _matching(name, res, shape, xf, "residual")
        res = _rows(res)
    be = _backend(xf)
    xr, wr = _rows(xf), _rows(weight)
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (xr, wr, bias, res)):
        y = _LinearAct.apply(xr, wr, bias, res, act, be)
    else:
        y = be.linear_fwd(xr, wr, bias, act, res)[0]
    return _wrapped(wrapper, y.view(shape), dim)


# ------------------------------------------------------------------------------------------------ norms around a block
class _NormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, y, out_weight, out_bias, gate, in_weight, in_bias, out_kind, in_kind, scale, eps, rows_per_gate, be):
        ctx.set_materialize_grads(False)
        ho, u, stats = be.norm_residual_fwd(h, y, out_weight, out_bias, gate, in_weight, in_bias, out_kind, in_kind, scale, eps, rows_per_gate, True)
        ctx.save_for_backward(h, y, out_weight, out_bias, gate, in_weight, in_bias, stats)
        ctx.meta, ctx.be = (out_kind, in_kind, scale, rows_per_gate), be
        return (ho, u) if ho is not None and u is not None else (ho if ho is not None else u)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        h, y, out_weight, out_bias, gate, in_weight, in_bias, stats = ctx.saved_tensors
        out_kind, in_kind, scale, rows_per_gate = ctx.meta
        gh = grads[0] if y is not None else None
        gu = grads[-1] if in_kind else None
        want = list(ctx.needs_input_grad[:7])
        if gh is None and gu is None:
            return (None,) * 13
        if h.shape[0] == 0:
            out = [torch.zeros_like(t) if w else None for t, w in zip((h, y, out_weight, out_bias, gate, in_weight, in_bias), want)]
        else:
            out = ctx.be.norm_residual_bwd(None if gh is None else _rows(gh), None if gu is None else _rows(gu), stats, h, y, out_weight, out_bias, gate, in_weight, in_bias,
                                           out_kind, in_kind, scale, rows_per_gate, want)
        return (*out, None, None, None, None, None, None)


def _gate(name, gate, hf, dim, packed):
    """(gate as (C,) or (samples, C), rows per gate): shapes (C,), or h's own with ones (broadcast over rows) and, for a gate per sample, h's
    first size; (C, 1, 1) as well for maps."""
    C = hf.shape[-1]
    gate = _plain(gate)
    if not isinstance(gate, torch.Tensor):
        raise TypeError(f"{name}: gate must be a tensor, got {type(gate).__name__}")
    if gate.dtype not in (hf.dtype, torch.float32) or gate.device != hf.device:
        raise TypeError(f"{name}: gate must be {hf.dtype} or float32 on {hf.device}, got {gate.dtype} on {gate.device}")
    shape = tuple(gate.shape)
    if dim == 1 and shape == (C, 1, 1):
        return gate.reshape(C).contiguous(), 0
    if shape == (C,):
        return gate.contiguous(), 0
    g = gate.permute(0, 2, 3, 1) if dim == 1 and gate.dim() == 4 else gate
    if g.dim() == hf.dim() and g.dim() >= 2 and g.shape[-1] == C and all(s == 1 for s in g.shape[1:-1]):
        if g.shape[0] == 1:
            return g.reshape(C).contiguous(), 0
        if g.shape[0] == hf.shape[0] and not packed:
            rows = hf.numel() // C
            return g.reshape(-1, C).contiguous(), rows // hf.shape[0] if rows else 0
    raise ValueError(f"{name}: gate must hold one value per channel ({C},) or per sample and channel, got {shape} for {tuple(hf.shape)} (features last)"
                     + ("; packed tiles are no samples" if packed else ""))


def norm_residual(h, y=None, *, out_norm: str = "none", out_weight=None, out_bias=None, gate=None, residual_scale: float = 1.0, in_norm: str = "none",
                  in_weight=None, in_bias=None, eps: float = 1e-6, dim: int = -1):
    """``(h', u)``: ``h' = residual_scale * h + gate * N_out(y)`` and ``u = N_in(h')`` over the features of each row.

    N is ``none``, ``rms`` (x / sqrt(mean x^2 + eps)) or ``layer`` (centred), times its weight plus its bias where given; the gate holds one
    value per channel, or per sample and channel.  Without ``y`` there is no block yet: h' is h itself.  Without ``in_norm`` u is None.
    Parameters in h's dtype or float32; up to 16384 channels.  u is formed from h' before its rounding."""
    name = "norm_residual"
    for k, what in ((out_norm, "out_norm"), (in_norm, "in_norm")):
        if k not in NORMS:
            raise ValueError(f"{name}: {what} must be one of {', '.join(NORMS)}, got {k!r}")
    if y is None and (out_norm != "none" or gate is not None or float(residual_scale) != 1.0):
        raise ValueError(f"{name}: out_norm, gate and residual_scale need a block's output y")
    if y is None and in_norm == "none":
        raise ValueError(f"{name}: nothing to do (neither y nor in_norm)")
    for norm, vecs, what in ((out_norm, (out_weight, out_bias), "out"), (in_norm, (in_weight, in_bias), "in")):
        if norm == "none" and any(v is not None for v in vecs):
            raise ValueError(f"{name}: {what}_weight / {what}_bias without {what}_norm")
    if not float(eps) >= 0.0:
        raise ValueError(f"{name}: eps must not be negative, got {eps}")
    hf, wrapper, dim = _argument(h, dim, name)
    C = hf.shape[-1]
    if C > MAX_NORM_CHANNELS:
        raise ValueError(f"{name}: at most {MAX_NORM_CHANNELS} channels, got {C}")
    packed = wrapper is not None and wrapper.is_blocks
    yf = None
    if y is not None:
        yf = _features(_plain(y), dim, name)
        _matching(name, yf, hf.shape, hf, "y")
    params = [_vector(name, p, C, hf, w) for p, w in ((out_weight, "out_weight"), (out_bias, "out_bias"), (in_weight, "in_weight"), (in_bias, "in_bias"))]
    rows_per_gate = 0
    if gate is not None:
        gate, rows_per_gate = _gate(name, gate, hf, dim, packed)
    params.insert(2, gate)
    if len({p.dtype for p in params if p is not None}) > 1:
        params = [None if p is None else p.float() for p in params]
    be = _backend(hf)
    hr, yr = _rows(hf), None if yf is None else _rows(yf)
    kinds = (NORMS[out_norm], NORMS[in_norm], float(residual_scale), float(eps), rows_per_gate)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (hr, yr, *params)):
        out = _NormResidual.apply(hr, yr, *params, *kinds, be)
        ho, u = out if isinstance(out, tuple) else ((out, None) if yr is not None else (None, out))
    else:
        ho, u, _ = be.norm_residual_fwd(hr, yr, *params, *kinds)
    back = lambda t: None if t is None else _wrapped(wrapper, t.view(hf.shape), dim)
    return (h if y is None else back(ho)), back(u)

"""Channel operators: what a residual network of row products is made of, on plain tensors and on packed tiles (NOT part of the reference's
API: an addition).

``linear_act``      y = act(x W^T + b) + residual: a 1x1 conv / linear layer with its whole epilogue in the product's kernel.
``norm_residual``   h' = residual_scale * h + gate * N_out(y),  u = N_in(h'): the norm after one block, the block's gate, the residual
                    stream and the norm before the next block in one pass.

Both work on rows of features: the last axis of a tensor (``dim=-1``, tokens), or axis 1 of a (N, C, H, W) map (``dim=1``, pixels), for which
channels-last memory is the free layout.  A packed or dense ``TensorWrapper`` is always read along axis 1 and gives a ``TensorWrapper``: rows
are independent of each other, so no halo, no transfer and no cache is involved, and skipped tiles keep their values when the result is
combined (in a frame sized for a ceiling of tiles every row is computed, the surplus ones out of whatever they hold, and gradients of
parameters are refused).  float32, float16 and bfloat16; sums, statistics, activations and everything between input and output in float32,
gradients too: nothing but a result is rounded to the tensors' type.  GPU tensors only.

Both are differentiable once with respect to every tensor argument, backward (a forward-mode tangent is refused).  Gradients of a captured
graph follow torch's rule for captured backward passes: warm up on the capturing stream, with no eager graph over the same leaves alive.  A small training step spends most of its
time on the host: capture it, or run it under ``torch.autograd.set_multithreading_enabled(False)`` (half the time uncaptured).  No call waits
for the device, and every result is run-to-run identical (sums are split and joined in a fixed order, no atomics)."""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
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


def _features(x, dim):
    """x with its features last."""
    return x.permute(0, 2, 3, 1) if dim == 1 else x


def _back(t, shape, dim):
    """Rows (rows, features) as a tensor of ``shape`` (its axis order, features anywhere), or None."""
    if t is None:
        return None
    return t.view(shape) if dim == -1 else t.view(shape[0], shape[2], shape[3], shape[1]).permute(0, 3, 1, 2)


def _result(x, shape, dim):
    """Memory for a result of ``shape`` whose features lie together.  Never a view: autograd lets results be modified in place (a ReLU)."""
    return x.new_empty(shape) if dim == -1 else torch.empty(shape, dtype=x.dtype, device=x.device, memory_format=torch.channels_last)


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
    if not isinstance(t, torch.Tensor) or t.shape != shape:
        raise ValueError(f"{name}: {what} must have the shape {tuple(shape)} (nothing is broadcast), got "
                         f"{tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__}")
    if t.dtype != like.dtype or t.device != like.device:
        raise TypeError(f"{name}: {what} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")


def _vector(name, p, n, like, what):
    """Per-channel parameter: n elements, the rows' dtype or float32."""
    if p is None:
        return None
    p = _plain(p)
    if not isinstance(p, torch.Tensor) or p.shape != (n,):
        raise ValueError(f"{name}: {what} must be a vector of {n} channels, got {tuple(p.shape) if isinstance(p, torch.Tensor) else p!r}")
    if (p.dtype != like.dtype and p.dtype != torch.float32) or p.device != like.device:
        raise TypeError(f"{name}: {what} must be {like.dtype} or float32 on {like.device}, got {p.dtype} on {p.device}")
    return p if p.is_contiguous() else p.contiguous()


def _argument(x, dim, name):
    """(plain tensor, its number of features, TensorWrapper or None, -1 or 1: where the features are)"""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name}: a tensor is needed, got {type(x).__name__}")
    wrapper = x if isinstance(x, TensorWrapper) and x.is_init else None
    x = _plain(x)
    if x.dtype not in _DTYPES:
        raise TypeError(f"{name}: float32, float16 or bfloat16 tensors, got {x.dtype}")
    n = x.dim()
    if wrapper is not None:
        dim = 1
    elif n and (dim == -1 or dim == n - 1):
        dim = -1
    if not (dim == -1 and n or dim == 1 and n == 4):
        raise ValueError(f"{name}: features are the last axis (dim=-1) or axis 1 of a (N, C, H, W) map (dim=1), got dim={dim} for shape {tuple(x.shape)}")
    if x.shape[dim] == 0:
        raise ValueError(f"{name}: no features in shape {tuple(x.shape)}")
    return x, x.shape[dim], wrapper, dim


def _surplus(wrapper):
    """Whether rows behind the executed tiles are there (a frame sized for a ceiling of tiles)."""
    return wrapper is not None and wrapper._dyn() is not None


def _refuse_sums(surplus, want, name):
    if surplus and any(want):
        raise NotImplementedError(f"{name}: gradients of parameters are sums over the executed tiles' rows, whose count only the device knows in this frame (block_graph=2)")


def _wrapped(out, wrapper):
    return out if out is None or wrapper is None else TensorWrapper._wrap_like(out, wrapper, wrapper.is_blocks)


def _watched(*tensors):
    """Whether the call has to go through autograd: for a backward pass, or because an argument carries a forward-mode tangent (which autograd
    refuses there: there is no forward-mode derivative, and a result without a tangent would say that it is zero)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if getattr(forward_ad, "_current_level", 0) >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                return True
    return False


def _first_order(fn):
    """``once_differentiable`` where a second derivative could be asked for at all (create_graph), else the function itself: its guard costs as
    much host time as a small product's launch."""
    guarded = once_differentiable(fn)

    def backward(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)

    return backward


# ------------------------------------------------------------------------------------------------ product
def _linear_rows(be, x, weight, bias, residual, act, dim, keep_z):
    """(y in the axis order of x, z, x's rows, the weight's rows)"""
    xr, wr = _rows(_features(x, dim)), _rows(weight if weight.dim() == 2 else weight.flatten(1))
    shape = list(x.shape)
    shape[dim] = wr.shape[0]
    y = _result(x, shape, dim)
    z = be.linear_fwd(xr, wr, bias, act, None if residual is None else _rows(_features(residual, dim)), keep_z, out=y)[1]
    return y, z, xr, wr


class _LinearAct(torch.autograd.Function):
    # (one node from argument to result: axis order, rows and their way back are inside)
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, dim, be, surplus):
        want = ctx.needs_input_grad
        y, z, xr, wr = _linear_rows(be, x, weight, bias, residual, act, dim, act != 0 and (want[0] or want[1] or want[2]))
        ctx.save_for_backward(xr if want[1] else None, wr if want[0] else None, z)
        ctx.meta = act, dim, be, x.shape, weight.shape, None if bias is None else bias.dtype, surplus
        return y

    @staticmethod
    @_first_order
    def backward(ctx, gy):
        xr, wr, z = ctx.saved_tensors
        act, dim, be, x_shape, w_shape, bias_dtype, surplus = ctx.meta
        want = ctx.needs_input_grad
        _refuse_sums(surplus, want[1:3], "linear_act")
        dx = dw = db = None
        if want[0] or want[1] or want[2]:
            dx, dw, db = be.linear_bwd(_rows(_features(gy, dim)), z, xr, wr, act, want, bias_dtype, saved=True)
            dx, dw = _back(dx, x_shape, dim), None if dw is None else dw.view(w_shape)
        return dx, dw, db, gy if want[3] else None, None, None, None, None


def linear_act(x, weight, bias=None, activation: str = "none", residual=None, dim: int = -1):
    """``act(x W^T + bias) + residual`` over the features of ``x``.

    weight (out, in), or (out, in, 1, 1) as a 1x1 conv keeps it, in x's dtype; bias (out,) in x's dtype or float32; activation one of
    ``none relu gelu gelu_tanh silu``; residual of the result's shape.  Any number of rows (none among them), any sizes, row strides as they
    come.  Under autograd the pre-activations are kept for the backward pass, in float32 for gelu, gelu_tanh and silu, and only the gradients
    themselves are rounded to x's dtype."""
    name = "linear_act"
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"{name}: activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    x, k, wrapper, dim = _argument(x, dim, name)
    weight = _plain(weight)
    if not isinstance(weight, torch.Tensor):
        raise TypeError(f"{name}: weight must be a tensor, got {type(weight).__name__}")
    n = weight.dim()
    if not (n == 2 or n == 4 and weight.shape[2] == weight.shape[3] == 1) or weight.shape[1] != k or weight.shape[0] == 0:
        raise ValueError(f"{name}: weight must be (out, {k}), got {tuple(weight.shape)}")
    if weight.dtype != x.dtype or weight.device != x.device:
        raise TypeError(f"{name}: weight must be {x.dtype} on {x.device}, got {weight.dtype} on {weight.device}")
    bias = _vector(name, bias, weight.shape[0], x, "bias")
    if residual is not None:
        residual = _plain(residual)
        shape = list(x.shape)
        shape[dim] = weight.shape[0]
        _matching(name, residual, torch.Size(shape), x, "residual")
    be = _backend(x)
    if _watched(x, weight, bias, residual):
        y = _LinearAct.apply(x, weight, bias, residual, act, dim, be, _surplus(wrapper))
    else:
        y = _linear_rows(be, x, weight, bias, residual, act, dim, False)[0]
    return _wrapped(y, wrapper)


# ------------------------------------------------------------------------------------------------ norms around a block
def _norm_rows(be, h, y, params, kinds, dim, keep_stats):
    """(h', u, stats, h's rows, y's rows); h', u in the axis order of h"""
    hr, yr = _rows(_features(h, dim)), None if y is None else _rows(_features(y, dim))
    wo, bo, gate, wi, bi = params
    ho, u, stats = None if y is None else _result(h, h.shape, dim), _result(h, h.shape, dim) if kinds[1] else None, None
    if hr.shape[0]:
        stats = be.norm_residual_fwd(hr, yr, wo, bo, None if gate is None else gate.view(-1), wi, bi, *kinds, keep_stats, out=(ho, u))[2]
    return ho, u, stats, hr, yr


class _NormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, y, out_weight, out_bias, gate, in_weight, in_bias, kinds, dim, be, surplus):
        ctx.set_materialize_grads(False)
        ho, u, stats, hr, yr = _norm_rows(be, h, y, (out_weight, out_bias, gate, in_weight, in_bias), kinds, dim, True)
        ctx.save_for_backward(hr, yr, out_weight, out_bias, gate, in_weight, in_bias, stats)
        ctx.meta = kinds, dim, be, h.shape, surplus
        return (ho, u) if ho is not None and u is not None else (ho if ho is not None else u)

    @staticmethod
    @_first_order
    def backward(ctx, *grads):
        h, y, out_weight, out_bias, gate, in_weight, in_bias, stats = ctx.saved_tensors
        (out_kind, in_kind, scale, _, rows_per_gate), dim, be, shape, surplus = ctx.meta
        gh = grads[0] if y is not None else None
        gu = grads[-1] if in_kind else None
        want = ctx.needs_input_grad[:7]
        if gh is None and gu is None:
            return (None,) * 11
        _refuse_sums(surplus, want[2:], "norm_residual")
        flat = None if gate is None else gate.view(-1)
        if h.shape[0] == 0:
            out = [torch.zeros_like(t) if w else None for t, w in zip((h, y, out_weight, out_bias, flat, in_weight, in_bias), want)]
        else:
            out = be.norm_residual_bwd(None if gh is None else _rows(_features(gh, dim)), None if gu is None else _rows(_features(gu, dim)), stats, h, y, out_weight, out_bias,
                                       flat, in_weight, in_bias, out_kind, in_kind, scale, rows_per_gate, want, saved=True)
        dh, dy, dwo, dbo, dg, dwi, dbi = out
        return (_back(dh, shape, dim), _back(dy, shape, dim), dwo, dbo, None if dg is None else dg.view(gate.shape), dwi, dbi, None, None, None, None)


def _gate(name, gate, h, C, dim, packed):
    """(gate, rows per gate): shapes (C,), (C, 1, 1) for maps, or h's own with ones (one gate for all rows) and, for a gate per sample, h's first size."""
    gate = _plain(gate)
    if not isinstance(gate, torch.Tensor):
        raise TypeError(f"{name}: gate must be a tensor, got {type(gate).__name__}")
    if (gate.dtype != h.dtype and gate.dtype != torch.float32) or gate.device != h.device:
        raise TypeError(f"{name}: gate must be {h.dtype} or float32 on {h.device}, got {gate.dtype} on {gate.device}")
    s = gate.shape
    gate = gate if gate.is_contiguous() else gate.contiguous()
    if s == (C,) or dim == 1 and s == (C, 1, 1):
        return gate, 0
    if len(s) == h.dim() >= 2 and s[dim] == C and gate.numel() == s[0] * C:
        if s[0] == 1:
            return gate, 0
        if s[0] == h.shape[0] and not packed:
            if s[0] > 65535:
                raise ValueError(f"{name}: gates for at most 65535 samples, got {s[0]}")
            return gate, h.numel() // gate.numel() if s[0] else 0
    raise ValueError(f"{name}: gate must hold one value per channel ({C},) or per sample and channel, got {tuple(s)} for {tuple(h.shape)}"
                     + ("; packed tiles are no samples" if packed else ""))


def norm_residual(h, y=None, *, out_norm: str = "none", out_weight=None, out_bias=None, gate=None, residual_scale: float = 1.0, in_norm: str = "none",
                  in_weight=None, in_bias=None, eps: float = 1e-6, dim: int = -1):
    """``(h', u)``: ``h' = residual_scale * h + gate * N_out(y)`` and ``u = N_in(h')`` over the features of each row.

    N is ``none``, ``rms`` (x / sqrt(mean x^2 + eps)) or ``layer`` (centred), times its weight plus its bias where given; the gate holds one
    value per channel, or per sample and channel.  Without ``y`` there is no block yet: h' is h itself.  Without ``in_norm`` u is None.
    Parameters in h's dtype or float32; up to 16384 channels.  u is formed from h' before its rounding."""
    name = "norm_residual"
    out_kind, in_kind, scale, eps = NORMS.get(out_norm), NORMS.get(in_norm), float(residual_scale), float(eps)
    if out_kind is None or in_kind is None:
        raise ValueError(f"{name}: out_norm and in_norm must be one of {', '.join(NORMS)}, got {out_norm!r}, {in_norm!r}")
    if y is None and (out_kind or gate is not None or scale != 1.0):
        raise ValueError(f"{name}: out_norm, gate and residual_scale need a block's output y")
    if y is None and not in_kind:
        raise ValueError(f"{name}: nothing to do (neither y nor in_norm)")
    if not out_kind and (out_weight is not None or out_bias is not None) or not in_kind and (in_weight is not None or in_bias is not None):
        raise ValueError(f"{name}: a norm's weight or bias without the norm")
    if not eps >= 0.0:
        raise ValueError(f"{name}: eps must not be negative, got {eps}")
    given = h
    h, C, wrapper, dim = _argument(h, dim, name)
    if C > MAX_NORM_CHANNELS:
        raise ValueError(f"{name}: at most {MAX_NORM_CHANNELS} channels, got {C}")
    if y is not None:
        y = _plain(y)
        _matching(name, y, h.shape, h, "y")
    rows_per_gate = 0
    if gate is not None:
        gate, rows_per_gate = _gate(name, gate, h, C, dim, wrapper is not None and wrapper.is_blocks)
    params = (_vector(name, out_weight, C, h, "out_weight"), _vector(name, out_bias, C, h, "out_bias"), gate, _vector(name, in_weight, C, h, "in_weight"),
              _vector(name, in_bias, C, h, "in_bias"))
    kind = None
    for p in params:
        if p is not None:
            if kind is None:
                kind = p.dtype
            elif p.dtype != kind:
                kind = False
    if kind is False:       # (the kernel takes one type of parameters)
        params = tuple(None if p is None else p.float() for p in params)
    be = _backend(h)
    kinds = (out_kind, in_kind, scale, eps, rows_per_gate)
    if _watched(h, y, *params):
        out = _NormResidual.apply(h, y, *params, kinds, dim, be, _surplus(wrapper))
        ho, u = out if isinstance(out, tuple) else ((out, None) if y is not None else (None, out))
    else:
        ho, u = _norm_rows(be, h, y, params, kinds, dim, False)[:2]
    return (given if y is None else _wrapped(ho, wrapper)), _wrapped(u, wrapper)

"""linear_act and norm_residual where their roundings, ranges and resources end."""
import itertools

import pytest
import torch

import channel_oracle as CO
from test_channel_ops import DT, _close, _norm_case, _rand, plain_backend  # noqa: F401  (a fixture)

SMOOTH = ("gelu", "gelu_tanh", "silu")


# ------------------------------------------------------------------------------------------------ gradients in 16 bits
@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("name", SMOOTH)
@pytest.mark.parametrize("M,K,N,size", [(130, 96, 72, 1.0), (513, 264, 200, 1.0), (1, 515, 1001, 1.0), (2049, 19, 130, 1.0), (33, 1000, 7, 1.0), (300, 512, 512, 2.0 ** -13),
                                        (1100, 1003, 1001, 1.0), (4100, 128, 1032, 2.0 ** 12)])
def test_gradients_round_once(dt, name, M, K, N, size):
    """Pre-activations and dz = dy act'(z) keep their bits until the gradient itself is rounded (``size``: of dy -- small ones lie among float16's
    subnormal numbers, large ones near its end)."""
    import blockcopy

    gen = torch.Generator().manual_seed(61)
    dtype = DT[dt]
    x, w, b = _rand(gen, M, K, dtype=dtype), _rand(gen, N, K, dtype=dtype, std=K ** -0.5), _rand(gen, N, dtype=dtype, std=0.3)
    gy = _rand(gen, M, N, dtype=dtype, std=size)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = blockcopy.linear_act(x, w, b, activation=name)
    want = CO.linear_gradients(x.detach(), w.detach(), b.detach(), name, gy)
    for k, got in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, gy)):
        v, bound = (t.cpu() for t in want[k])
        # (a value beyond the type's largest number rounds to an infinity of its sign; at the border, within the bound, either is right)
        over = v.abs() + bound > torch.finfo(dtype).max
        _close(torch.where(over, v, got.double().cpu()), v, bound, (dt, M, K, N, name, k))
        assert bool((got.double().cpu() * v.sign() >= v.abs() - bound)[over].all()), (dt, M, K, N, name, k)


@pytest.mark.gpu
def test_gradients_round_once_in_every_product_shape():
    """The large tiles, slices and partial steps of both products: the share of the error that is not the result's own rounding (which alone
    gives the ratio 1) is at most a tenth."""
    import blockcopy

    sizes = [(8192, 1032, 2056, 1.0), (4100, 4104, 72, 1.0), (72, 4104, 4104, 1.0), (600, 4000, 4000, 1.0), (16384, 136, 264, 1.0), (1500, 1002, 1004, 1.0),
             (16384, 136, 264, 2.0 ** -18)]        # (the last: dy and dz among float16's subnormal numbers)
    for dtype, (M, K, N, size), name in itertools.product((torch.float16, torch.bfloat16), sizes, ("gelu", "silu")):
        gen = torch.Generator(device="cuda").manual_seed(62)
        r = lambda *s, std=1.0: (torch.randn(s, generator=gen, device="cuda") * std).to(dtype)
        x, w, b, gy = r(M, K).requires_grad_(True), r(N, K, std=K ** -0.5).requires_grad_(True), r(N).requires_grad_(True), r(M, N, std=size)
        got = torch.autograd.grad(blockcopy.linear_act(x, w, b, activation=name), [x, w, b], gy)
        d = lambda t: t.detach().double()
        dz = d(gy) * CO.act(d(x) @ d(w).t() + d(b), name)[1]
        for k, g, e in zip(("dx", "dw", "db"), got, (dz @ d(w), dz.t() @ d(x), dz.sum(0))):
            own = float((e.to(dtype).double() - e).norm())
            assert float((g.double() - e).norm()) <= 1.1 * own, (dtype, M, K, N, name, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
def test_relu_passes_what_is_above_zero(dt):
    """A pre-activation above zero that is too small for the tensors' type still passes its gradient; one below or at zero none."""
    import blockcopy

    tiny = 2.0 ** -14 if dt == "f16" else 2.0 ** -40
    x = torch.tensor([[tiny], [-tiny], [0.0]], dtype=DT[dt], device="cuda").requires_grad_(True)
    w = torch.full((9, 1), tiny, dtype=DT[dt], device="cuda").requires_grad_(True)
    (gx,) = torch.autograd.grad(blockcopy.linear_act(x, w, activation="relu"), [x], torch.ones(3, 9, dtype=DT[dt], device="cuda"))
    assert torch.equal(gx, torch.tensor([[9 * tiny], [0.0], [0.0]], dtype=DT[dt], device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
def test_infinite_gradients_keep_their_sign(dt):
    """An infinity or NaN in dy reaches its own row of dx and its own column's row of dw, as such."""
    import blockcopy

    gen = torch.Generator().manual_seed(63)
    x, w = _rand(gen, 40, 24, dtype=DT[dt]), _rand(gen, 16, 24, dtype=DT[dt]).abs() + 0.5
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    gy = _rand(gen, 40, 16, dtype=DT[dt])
    run = lambda g: torch.autograd.grad(blockcopy.linear_act(x, w, activation="silu"), [x, w], g)
    clean = run(gy)
    gy = gy.clone()
    with torch.no_grad():
        z = x.double() @ w.double().t()
    gy[3, 5], gy[9, 7] = float("inf"), float("nan")
    dx, dw = run(gy)
    sign = CO.act(z[3, 5], "silu")[1].sign()
    assert bool((dx[3] == float("inf") * sign).all()) and bool(dx[9].isnan().all())
    keep, cols = [i for i in range(40) if i not in (3, 9)], [i for i in range(16) if i not in (5, 7)]
    assert torch.equal(dx[keep], clean[0][keep]) and torch.equal(dw[cols], clean[1][cols])
    assert bool((dw[5] == float("inf") * sign * x[3].sign()).all()) and bool(dw[7].isnan().all())


# ------------------------------------------------------------------------------------------------ activations far out
@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("name", CO.ACTS)
def test_derivatives_far_out(dt, name):
    """act'(z) beyond the range that the exponentials cover.  One input, one weight of 1, dy = 1: the data gradient is act'(z), rounded once.  32
    roundings of its own, (z^2 + 2 |z|) U from the exponent's roundings, and where a sigmoid or exponential lies below float32's smallest normal
    number 2^-126 it may be 0: an error of 2^-126 times what it is multiplied by, at most (1 + |z|)^3."""
    import blockcopy

    z = torch.tensor([s * v for v in (0.5, 20.0, 40.0, 63.0, 64.0, 65.0, 80.0, 86.0, 90.0, 110.0, 127.0, 128.0, 130.0, 200.0, 1000.0, 60000.0) for s in (1, -1)], dtype=torch.float64)
    x = z.to(DT[dt]).cuda()[:, None].requires_grad_(True)
    w = torch.ones(1, 1, dtype=DT[dt], device="cuda")
    (gx,) = torch.autograd.grad(blockcopy.linear_act(x, w, activation=name), [x], torch.ones(len(z), 1, dtype=DT[dt], device="cuda"))
    z = x.detach().double().cpu()
    d = CO.act(z, name)[1]
    inner = {"gelu": z * z, "gelu_tanh": 1.6 * z.abs() * (1 + 0.045 * z * z)}.get(name, z.abs())
    err = 32 * CO.U * d.abs() + 2 * inner.clamp_max(200) * CO.U * d.abs() + 2.0 ** -126 * (1 + z.abs().clamp_max(128)) ** 3 + 32 * CO.U * (z.abs() < 10)
    _close(gx, d, CO.rounded(d, err, DT[dt]), (dt, name))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
def test_tails_of_gelu(dt):
    """gelu(z) = z Phi(z) keeps its relative precision where Phi is small: Phi's own error (2^-19 in 16-bit types, 64 U in float32, besides the
    exponent's: z^2 / 2 off by at most 4 roundings) times the value, never 1 - (1 - Phi)."""
    import blockcopy

    z = -torch.linspace(0.01, 12.9, 700, dtype=torch.float64)
    x = z.to(DT[dt]).cuda()[:, None]
    y = blockcopy.linear_act(x, torch.ones(1, 1, dtype=DT[dt], device="cuda"), activation="gelu")
    z = x.double().cpu()
    a = CO.act(z, "gelu")[0]
    err = a.abs() * ((64 * CO.U if dt == "f32" else 2.0 ** -19) + 2 * z * z * CO.U)
    _close(y, a, CO.rounded(a, err, DT[dt]), dt)


# ------------------------------------------------------------------------------------------------ refusals
@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused_by_linear_act(plain_backend, which, grad):  # noqa: F811
    """There is no forward-mode derivative: a dual argument raises, whichever it is, instead of losing its tangent."""
    import blockcopy
    import torch.autograd.forward_ad as fw

    args = [torch.randn(3, 4), torch.randn(5, 4), torch.randn(5), torch.randn(3, 5)]
    call = lambda a: blockcopy.linear_act(a[0], a[1], a[2], activation="silu", residual=a[3])
    with torch.set_grad_enabled(grad):
        with fw.dual_level():
            assert torch.equal(call(args), call(args))       # (no tangent: as ever)
            args[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
            with pytest.raises((RuntimeError, NotImplementedError)):
                call(args)
        with pytest.raises((RuntimeError, NotImplementedError)):
            plain = [fw.unpack_dual(a).primal if isinstance(a, torch.Tensor) else a for a in args]
            torch.func.jvp(lambda t: call([t if i == which else p for i, p in enumerate(plain)]), (plain[which],), (torch.ones_like(plain[which]),))


@pytest.mark.parametrize("which", range(7))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused_by_norm_residual(plain_backend, which, grad):  # noqa: F811
    import blockcopy
    import torch.autograd.forward_ad as fw

    args = [torch.randn(3, 4), torch.randn(3, 4), *(torch.randn(4) for _ in range(5))]
    call = lambda a: blockcopy.norm_residual(a[0], a[1], out_norm="rms", out_weight=a[2], out_bias=a[3], gate=a[4], in_norm="layer", in_weight=a[5], in_bias=a[6])
    with torch.set_grad_enabled(grad), fw.dual_level():
        call(args)
        args[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(args)


def test_parameter_gradients_of_a_frame_with_surplus_tiles_are_refused(plain_backend):  # noqa: F811
    """In a frame sized for a ceiling of tiles the rows behind the executed ones hold anything: a sum over all rows is no gradient.  The data
    gradients, row by row, are those of the rows."""
    import blockcopy

    def frame(dyn):
        t = blockcopy.to_tensorwrapper(torch.randn(2, 6, 8, 8).contiguous(memory_format=torch.channels_last))
        t.process_temporal_features(None)
        t._is_blocks = True
        t._features.dyn = (torch.tensor([1]), 2) if dyn else None
        return t

    w, v = torch.randn(6, 6, requires_grad=True), torch.randn(6, requires_grad=True)
    for dyn in (False, True):
        calls = [lambda: blockcopy.linear_act(frame(dyn), w), lambda: blockcopy.linear_act(frame(dyn), w.detach(), v), lambda: blockcopy.norm_residual(frame(dyn), frame(dyn), gate=v)[0],
                 lambda: blockcopy.norm_residual(frame(dyn), in_norm="rms", in_weight=v)[1]]
        for call in calls:
            out = call()._plain()
            if dyn:
                with pytest.raises(NotImplementedError):
                    out.sum().backward()
            else:
                out.sum().backward()


# ------------------------------------------------------------------------------------------------ many gates
@pytest.mark.parametrize("M,C,rpg", [(65535, 4096, 1), (65535 * 2, 1024, 2), (65528, 1024, 8), (65535, 16384, 1), (65535, 16, 1), (60000, 9000, 3), (4200, 48, 2)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_workspace_of_many_gates(M, C, rpg, dtype):
    """The backward pass asks for no more than the size of one of its tensors, or 32 MB."""
    import blockcopy.backend as bk

    assert bk.load_library().bc_norm_residual_bwd_workspace(M, C, rpg, dtype) <= max(M * C * (4 if dtype == 0 else 2), 32 << 20) + 8 * M


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("M,C,groups", [(20000, 64, 20000), (30003, 33, 30003), (9000, 200, 4500), (9002, 201, 4501), (2400, 1030, 1200), (900, 4096, 450), (600, 8192, 300), (300, 9000, 100),
                                        (60, 16384, 60), (6000, 520, 2000)])
def test_many_gates(dt, M, C, groups):
    """Gates of few rows each: every gradient."""
    _norm_case(dt, M, C, "layer", "rms", gate="sample", groups=groups, seed=71)
    _norm_case(dt, M, C, "none", "layer", gate="sample", groups=groups, seed=72, bias=False)


@pytest.mark.gpu
@pytest.mark.parametrize("M,C,groups", [(20000, 64, 20000), (300, 9000, 100), (9002, 201, 4501)])
def test_many_gates_each_gradient_alone(M, C, groups):
    import blockcopy

    gen = torch.Generator().manual_seed(73)
    dtype, R = torch.bfloat16, M // groups
    ts = [_rand(gen, groups, R, C, dtype=dtype), _rand(gen, groups, R, C, dtype=dtype), *(_rand(gen, C, dtype=dtype, mean=1.0, std=0.2) for _ in range(2)),
          _rand(gen, groups, 1, C, dtype=dtype), *(_rand(gen, C, dtype=dtype, mean=1.0, std=0.2) for _ in range(2))]
    gs = [_rand(gen, groups, R, C, dtype=dtype) for _ in range(2)]

    def grads(live):
        a = [t.clone().requires_grad_(i in live) for i, t in enumerate(ts)]
        out = blockcopy.norm_residual(a[0], a[1], out_norm="layer", out_weight=a[2], out_bias=a[3], gate=a[4], in_norm="rms", in_weight=a[5], in_bias=a[6])
        return torch.autograd.grad(out, [a[i] for i in live], gs)

    full = grads(range(7))
    for i in range(7):
        assert torch.equal(grads([i])[0], full[i]), i
    assert all(torch.equal(p, q) for p, q in zip(full, grads(range(7))))


# ------------------------------------------------------------------------------------------------ more rows than one step of every workgroup
def _rows_at_once(C):
    """Rows that one step of a whole launch takes at most, and rows that any launch of the backward pass takes in one step: a row of up to 512
    channels is a power of two of lanes with eight channels each, 256 lanes a workgroup; up to 1024 two rows share a workgroup; beyond one."""
    lanes = 1
    while lanes < 64 and 8 * lanes < C:
        lanes *= 2
    per = 256 // lanes if C <= 512 else 2 if C <= 1024 else 1
    return (1280 if C <= 2048 else 512) * per, 256 * per


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("C", [5, 40, 200, 500, 1001, 1024, 1500, 2048, 2100, 4096, 4100, 8192, 8200, 9001])
def test_norm_rows_of_later_steps(dt, C):
    """Workgroups that take four rows and more, the last step ragged: every row's results and gradients have the bits that the same row has in a
    call where each workgroup takes one step, and the column sums are those of all rows."""
    import blockcopy

    most, once = _rows_at_once(C)
    M = 3 * most + most // 3 + 1
    assert M > 3 * most
    gen = torch.Generator(device="cuda").manual_seed(81)
    dtype = DT[dt]
    r = lambda *s, std=1.0, mean=0.0, t=dtype: (torch.randn(s, generator=gen, device="cuda") * std + mean).to(t)
    h, y, gh, gu = r(M, C, mean=0.3), r(M, C, std=0.7), r(M, C), torch.randint(-3, 4, (M, C), generator=gen, device="cuda").to(dtype)
    ps = [r(C, std=0.2, mean=1.0, t=torch.float32) for _ in range(5)]
    names = ("out_weight", "out_bias", "gate", "in_weight", "in_bias")

    def run(rows):
        a = [t[rows].clone().requires_grad_(True) for t in (h, y)] + [p.clone().requires_grad_(True) for p in ps]
        out = blockcopy.norm_residual(a[0], a[1], out_norm="layer", in_norm="layer", **dict(zip(names, a[2:])))
        return [*(o.detach() for o in out), *torch.autograd.grad(out, a, (gh[rows], gu[rows]))]

    whole = run(slice(0, M))
    sums = [torch.zeros(C, dtype=torch.float64, device="cuda") for _ in range(5)]
    for m in range(0, M, once):
        part = run(slice(m, min(M, m + once)))
        for k in range(4):
            assert torch.equal(whole[k][m:m + once], part[k]), (C, k, m)
        for s, p in zip(sums, part[4:]):
            s += p.double()
    assert torch.equal(whole[8].double(), gu.double().sum(0))       # (whole numbers: d in_bias is exact)
    # the other sums: both sides add at most 200 partial results of a column in a row, of terms no larger than these
    n = lambda x: (x - x.mean(-1, keepdim=True)) / (x.var(-1, keepdim=True, unbiased=False) + 1e-6).sqrt() if C > 1 else x * 0
    ny, nh = n(y.double()).abs(), n(whole[0].double()).abs() * 1.02 + 0.02
    sd = whole[0].double().std(-1, keepdim=True)
    q = gu.double().abs() * ps[3].double().abs()
    g = gh.double().abs() + (q + q.mean(-1, keepdim=True) + nh * (q * nh).mean(-1, keepdim=True)) / sd.clamp_min(1e-3) * 1.02
    gate = ps[2].double().abs()
    sizes = [(g * gate * ny).sum(0), (g * gate).sum(0), (g * (ny * ps[0].double().abs() + ps[1].double().abs())).sum(0), (gu.double().abs() * nh).sum(0)]
    for k, (s, size) in enumerate(zip(sums, sizes)):
        over = (whole[4 + k].double() - s).abs() - 2 * 200 * CO.U * size
        assert bool((over <= 0).all()), (C, names[k], float(over.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("C,groups", [(40, 3), (500, 2), (1001, 3), (2048, 5), (4100, 2), (9001, 3)])
def test_norm_long_gate_groups(dt, C, groups):
    """A gate per sample of many rows: whole numbers without norms, so that every gradient is exact."""
    import blockcopy

    R = 3 * _rows_at_once(C)[0] // groups + 7
    gen = torch.Generator(device="cuda").manual_seed(83)
    pick = lambda *s: torch.randint(-2, 3, s, generator=gen, device="cuda").to(DT[dt])
    h, y, gh = pick(groups, R, C).requires_grad_(True), pick(groups, R, C).requires_grad_(True), pick(groups, R, C)
    gate = torch.randint(-2, 3, (groups, 1, C), generator=gen, device="cuda").float().requires_grad_(True)
    ho, _ = blockcopy.norm_residual(h, y, gate=gate, residual_scale=2.0)
    assert torch.equal(ho.double(), 2 * h.double() + gate.double() * y.double())
    dh, dy, dg = torch.autograd.grad(ho, [h, y, gate], gh)
    assert torch.equal(dh.double(), 2 * gh.double()) and torch.equal(dy.double(), gate.double() * gh.double())
    assert torch.equal(dg.double(), (gh.double() * y.double()).sum(1, keepdim=True))


@pytest.mark.gpu
def test_gradient_offsets_beyond_32_bits():
    """More than 2^31 elements of dz: the far rows' pre-activations and both parts of dz lie at their own places."""
    import blockcopy

    K, N, far = 24, 1032, 300
    M = (1 << 31) // N + far
    gen = torch.Generator().manual_seed(91)
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[-far:] = _rand(gen, far, K, dtype=torch.bfloat16)
    w, b = _rand(gen, N, K, dtype=torch.bfloat16, std=K ** -0.5), _rand(gen, N, dtype=torch.bfloat16, std=0.3)
    gy = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    gy[-far:] = _rand(gen, far, N, dtype=torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = blockcopy.linear_act(x, w, b, activation="silu")
    dx, dw, db = torch.autograd.grad(y, leaves, gy)
    # (the other rows' terms are zeros: they change no bound)
    want = CO.linear_gradients(x.detach()[-far:], w.detach(), b.detach(), "silu", gy[-far:])
    _close(dx[-far:], *want["dx"], "dx")
    _close(dw, *want["dw"], "dw")
    _close(db, *want["db"], "db")
    assert not bool(dx[:-far].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("name", SMOOTH)
def test_infinite_operands_of_gradients(dt, name):
    """An infinity in a row of x or w makes the gradients that it is multiplied into what the products say: infinite with the sign of dz, NaN where dz
    is zero -- in those places only."""
    import blockcopy

    gen = torch.Generator().manual_seed(93)
    x, w = _rand(gen, 70, 40, dtype=DT[dt]), _rand(gen, 24, 40, dtype=DT[dt])
    gy = _rand(gen, 70, 24, dtype=DT[dt])
    x[9, 3] = float("inf")
    run = lambda a, b: torch.autograd.grad(blockcopy.linear_act(a.requires_grad_(True), b.requires_grad_(True), activation=name), [a, b], gy)
    dx, dw = run(x.clone(), w.clone())
    # row 9: z = +-inf, act' = 1 or 0, dz = gy or +-0
    up = w[:, 3] > 0
    want = torch.where(up, gy[9].sign() * float("inf"), torch.full_like(gy[9], float("nan")))
    assert torch.equal(dw[up, 3], want[up]) and bool(dw[~up, 3].isnan().all())
    keep = [i for i in range(40) if i != 3]
    assert bool(dw[:, keep].isfinite().all()) and bool(dx.isfinite().all())
    x[9, 3], w[7, 5] = 0.0, float("inf")
    dx, dw = run(x.clone(), w.clone())
    # column 7 of z = +-inf by the sign of x[:, 5]
    up = x[:, 5] > 0
    assert torch.equal(dx[up, 5], gy[up, 7].sign() * float("inf")) and bool(dx[~up, 5].isnan().all())
    keep = [i for i in range(40) if i != 5]
    assert bool(dx[:, keep].isfinite().all()) and bool(dw.isfinite().all())

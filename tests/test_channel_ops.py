"""linear_act and norm_residual: refusals, host logic and gradients' formulas on the CPU; the kernels against the 64-bit definitions on the GPU,
within bounds that count their roundings (channel_oracle.py)."""
import itertools

import pytest
import torch

import channel_oracle as CO

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class PlainBackend:
    """What the host logic is tested with: the backend's channel operators in 64 bits with torch."""

    name = "plain"

    @staticmethod
    def _put(out, rows):
        if out is None or rows is None:
            return rows
        (out.permute(0, 2, 3, 1) if out.dim() == 4 and out.numel() and out.stride(1) == 1 else out).view(rows.shape).copy_(rows)
        return out

    def linear_fwd(self, x, w, b=None, act=0, res=None, keep_z=False, out=None):
        z = x.double() @ w.double().t() + (0 if b is None else b.double())
        y = CO.act(z, CO.ACTS[act])[0] + (0 if res is None else res.double())
        return self._put(out, y.to(x.dtype)), z.to(x.dtype) if keep_z else None

    def linear_bwd(self, gy, z, x, w, act, want, bias_dtype=None, saved=False):
        dz = gy.double() * (1 if act == 0 else CO.act(z.double(), CO.ACTS[act])[1])
        return ((dz @ w.double()).to(gy.dtype) if want[0] else None, (dz.t() @ x.double()).to(gy.dtype) if want[1] else None,
                dz.sum(0).to(bias_dtype or gy.dtype) if want[2] else None)

    @staticmethod
    def _norm(h, y, wo, bo, gate, wi, bi, out_kind, in_kind, scale, eps, rpg):
        kinds = ("none", "rms", "layer")
        gate = gate if gate is None or not rpg else gate.view(-1, h.shape[1])
        return CO.norm_residual(h, y, {"wo": wo, "bo": bo, "wi": wi, "bi": bi}, gate, scale, kinds[out_kind], kinds[in_kind], eps, rpg)

    def norm_residual_fwd(self, h, y, wo, bo, gate, wi, bi, out_kind, in_kind, scale, eps, rpg=0, keep_stats=False, out=(None, None)):
        args = [None if t is None else t.double() for t in (h, y, wo, bo, gate, wi, bi)]
        ho, u = self._norm(*args, out_kind, in_kind, scale, eps, rpg)
        stats = torch.full((h.shape[0], 4), eps) if keep_stats else None
        return None if y is None else self._put(out[0], ho.to(h.dtype)), None if u is None else self._put(out[1], u.to(h.dtype)), stats

    def norm_residual_bwd(self, gh, gu, stats, h, y, wo, bo, gate, wi, bi, out_kind, in_kind, scale, rpg, want, saved=False):
        src = (h, y, wo, bo, gate, wi, bi)
        args = [None if t is None else t.detach().double().requires_grad_(True) for t in src]
        with torch.enable_grad():
            ho, u = self._norm(*args, out_kind, in_kind, scale, float(stats[0, 0]), rpg)
        outs = [(o, g) for o, g in ((ho, gh), (u, gu)) if g is not None]
        leaves = [a for a, w in zip(args, want) if w]
        got = iter(torch.autograd.grad([o for o, _ in outs], leaves, [g.double() for _, g in outs], allow_unused=True))
        return tuple((lambda g, s: torch.zeros_like(s) if g is None else g.to(s.dtype))(next(got), s) if w else None for s, w in zip(src, want))


@pytest.fixture()
def plain_backend():
    import blockcopy.backend as bk

    prev = bk.set_backend(PlainBackend())
    yield
    bk.set_backend(prev)


def _close(got, want, bound, what):
    got = got.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    over = (got - want.cpu()).abs() - bound.cpu()
    assert bool((over <= 0).all()), (what, "largest excess", float(over.max()), "at", int(over.argmax()), "error", float((got - want.cpu()).abs().max()))


# ------------------------------------------------------------------------------------------------ CPU: refusals and host logic
def test_refusals_of_linear_act(plain_backend):
    import blockcopy

    x, w = torch.randn(3, 8), torch.randn(5, 8)
    bad = [(ValueError, lambda: blockcopy.linear_act(x, w, activation="tanh")), (ValueError, lambda: blockcopy.linear_act(x, torch.randn(5, 7))),
           (ValueError, lambda: blockcopy.linear_act(x, torch.randn(8))), (ValueError, lambda: blockcopy.linear_act(x, w, torch.randn(4))),
           (ValueError, lambda: blockcopy.linear_act(x, w, torch.randn(1, 5))), (ValueError, lambda: blockcopy.linear_act(x, w, residual=torch.randn(1, 5))),
           (ValueError, lambda: blockcopy.linear_act(x, w, residual=torch.randn(5))), (TypeError, lambda: blockcopy.linear_act(x, w.half())),
           (TypeError, lambda: blockcopy.linear_act(x, w, torch.randn(5).half())), (TypeError, lambda: blockcopy.linear_act(x, w, residual=torch.randn(3, 5).half())),
           (TypeError, lambda: blockcopy.linear_act(x.double(), w.double())), (TypeError, lambda: blockcopy.linear_act(x.long(), w)),
           (ValueError, lambda: blockcopy.linear_act(x, w, dim=0)), (ValueError, lambda: blockcopy.linear_act(torch.randn(2, 8, 4), w, dim=1)),
           (ValueError, lambda: blockcopy.linear_act(torch.tensor(1.0), w)), (ValueError, lambda: blockcopy.linear_act(torch.randn(3, 0), torch.randn(5, 0))),
           (ValueError, lambda: blockcopy.linear_act(x, torch.randn(0, 8))), (ValueError, lambda: blockcopy.linear_act(x, torch.randn(5, 8, 3, 3))),
           (TypeError, lambda: blockcopy.linear_act([1.0], w))]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def test_refusals_of_norm_residual(plain_backend):
    import blockcopy

    h, y, v = torch.randn(6, 8), torch.randn(6, 8), torch.ones(8)
    f = blockcopy.norm_residual
    bad = [(ValueError, lambda: f(h)), (ValueError, lambda: f(h, y, out_norm="batch")), (ValueError, lambda: f(h, in_norm="rms", gate=v)),
           (ValueError, lambda: f(h, in_norm="rms", residual_scale=0.5)), (ValueError, lambda: f(h, out_norm="rms", in_norm="rms")),
           (ValueError, lambda: f(h, y, out_weight=v)), (ValueError, lambda: f(h, y, in_bias=v)), (ValueError, lambda: f(h, torch.randn(6, 7))),
           (ValueError, lambda: f(h, torch.randn(1, 8))), (TypeError, lambda: f(h, y.half())), (ValueError, lambda: f(h, y, gate=torch.ones(7))),
           (ValueError, lambda: f(h, y, gate=torch.ones(3, 8))), (TypeError, lambda: f(h, y, gate=v.half())), (TypeError, lambda: f(h, y, gate=0.5)),
           (ValueError, lambda: f(h, y, out_norm="rms", out_weight=torch.ones(1))), (ValueError, lambda: f(h, y, in_norm="rms", eps=-1.0)),
           (ValueError, lambda: f(h, y, in_norm="rms", eps=float("nan"))), (ValueError, lambda: f(torch.randn(1, 16385), in_norm="rms")),
           (TypeError, lambda: f(h.double(), in_norm="rms")), (ValueError, lambda: f(torch.randn(2, 3, 8), torch.randn(2, 3, 8), gate=torch.ones(2, 3, 8))),
           (ValueError, lambda: f(h, y, dim=0)), (ValueError, lambda: f(torch.randn(65536, 1), torch.randn(65536, 1), gate=torch.ones(65536, 1)))]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def test_no_cpu_path():
    """The product has one backend: host tensors are refused, not computed elsewhere."""
    import blockcopy
    from blockcopy.backend import BlockCopyBackendError

    with pytest.raises(BlockCopyBackendError):
        blockcopy.linear_act(torch.randn(2, 4), torch.randn(3, 4))
    with pytest.raises(BlockCopyBackendError):
        blockcopy.norm_residual(torch.randn(2, 4), in_norm="rms")


def test_c_entries_validate_before_any_device_call():
    import blockcopy.backend as bk

    lib, N = bk.load_library(), None
    lin = lambda *, y=256, x=256, w=256, res=N, M=4, n=8, k=16, ldx=16, ldw=16, ldr=0, act=0, dt=0, ws=N, wsb=0: lib.bc_linear_fwd(
        y, N, x, w, N, res, M, n, k, ldx, ldw, ldr, act, dt, 0, ws, wsb, N)
    assert lin(M=0) == 0 and lin(M=-1) == -2 and lin(n=0) == -2 and lin(k=0) == -2 and lin(dt=3) == -3 and lin(act=5) == -2 and lin(act=-1) == -2
    assert lin(ldx=15) == -2 and lin(ldw=15) == -2 and lin(res=256, ldr=7) == -2 and lin(y=N) == -1 and lin(x=N) == -1 and lin(w=N) == -1
    assert lin(x=258) == -5 and lin(M=1 << 31) == -4
    need = lib.bc_linear_fwd_workspace(100, 8, 1 << 16, 0)
    assert need > 0 and lin(M=100, k=1 << 16, ldx=1 << 16, ldw=1 << 16) == -1 and lin(M=100, k=1 << 16, ldx=1 << 16, ldw=1 << 16, ws=256, wsb=need - 1) == -2
    bwd = lambda *, dx=256, dw=256, db=256, gy=256, z=256, x=256, w=256, M=4, n=8, k=16, ldg=8, ldx=16, ldw=16, act=1, dt=0, ws=256, wsb=1 << 30: lib.bc_linear_bwd(
        dx, dw, db, gy, z, x, w, M, n, k, ldg, ldx, ldw, act, dt, 0, ws, wsb, N)
    assert bwd(M=0) == -2 and bwd(gy=N) == -1 and bwd(z=N) == -1 and bwd(x=N) == -1 and bwd(w=N) == -1 and bwd(ldg=7) == -2 and bwd(ws=N) == -1
    assert bwd(wsb=lib.bc_linear_bwd_workspace(4, 8, 16, 1, 0) - 1) == -2 and bwd(ws=300) == -5 and bwd(dt=-1) == -3
    fwd = lambda *, ho=256, u=256, h=256, y=256, gate=N, M=6, C=8, ldh=8, ldy=8, rpg=0, ok=1, ik=1, dt=0, stats=N: lib.bc_norm_residual_fwd(
        ho, u, stats, h, y, N, N, gate, N, N, M, C, ldh, ldy, rpg, 1.0, 1e-6, ok, ik, dt, 0, N)
    assert fwd(M=0) == 0 and fwd(C=16385) == -2 and fwd(C=0) == -2 and fwd(ok=3) == -2 and fwd(ik=-1) == -2 and fwd(dt=4) == -3 and fwd(ldh=7) == -2
    assert fwd(M=65536, gate=256, rpg=1) == -4 and lin(M=1 << 30, n=1 << 30) == -4
    assert fwd(rpg=2) == -2 and fwd(gate=256, rpg=4) == -2 and fwd(y=N) == -2 and fwd(y=N, ok=0, ik=0) == -2 and fwd(h=N) == -1 and fwd(u=N) == -1
    assert fwd(stats=264) == -5 and fwd(h=257) == -5 and fwd(M=1 << 31) == -4
    nb = lambda *, dh=256, dy=256, dwo=256, stats=256, h=256, y=256, M=6, C=8, ldh=8, ws=256, wsb=1 << 30: lib.bc_norm_residual_bwd(
        dh, dy, dwo, N, N, N, N, 256, N, stats, h, y, N, N, N, N, M, C, ldh, 8, 8, 8, 0, 1.0, 1, 0, 0, 0, ws, wsb, N)
    assert nb(M=0) == -2 and nb(stats=N) == -1 and nb(h=N) == -1 and nb(ws=N) == -1 and nb(wsb=3) == -2 and nb(ldh=4) == -2 and nb(stats=260) == -5


@pytest.mark.parametrize("name", CO.ACTS)
def test_plain_gradients_against_differences(name):
    """The oracle's activation derivatives are those of its activations (central differences in 64 bits: error h^2 / 6 |act'''| + 1e-16 / h)."""
    z = torch.linspace(-6.03, 6.01, 301, dtype=torch.float64)
    h = 1e-5
    fd = (CO.act(z + h, name)[0] - CO.act(z - h, name)[0]) / (2 * h)
    assert float((fd - CO.act(z, name)[1]).abs().max()) < 1e-8


@pytest.mark.parametrize("name,dim,bias,res", [(a, d, b, r) for a, d, (b, r) in itertools.product(("none", "gelu"), (-1, 1), ((True, True), (False, False)))])
def test_linear_act_host_logic(plain_backend, name, dim, bias, res):
    """Axis order, weight shapes and autograd wiring, against torch's own ops."""
    import blockcopy

    g = torch.Generator().manual_seed(1)
    x = torch.randn((2, 6, 3, 5) if dim == 1 else (2, 3, 5, 6), generator=g).requires_grad_(True)
    w = torch.randn((4, 6, 1, 1) if dim == 1 else (4, 6), generator=g).requires_grad_(True)
    b = torch.randn(4, generator=g).requires_grad_(True) if bias else None
    r = torch.randn((2, 4, 3, 5) if dim == 1 else (2, 3, 5, 4), generator=g).requires_grad_(True) if res else None
    y = blockcopy.linear_act(x, w, b, activation=name, residual=r, dim=dim)
    ref = torch.nn.functional.conv2d(x, w, b) if dim == 1 else torch.nn.functional.linear(x, w, b)
    ref = (torch.nn.functional.gelu(ref) if name == "gelu" else ref) + (0 if r is None else r)
    assert y.shape == ref.shape and torch.allclose(y, ref, atol=1e-5)
    gy = torch.randn(y.shape, generator=g)
    leaves = [t for t in (x, w, b, r) if t is not None]
    for got, want in zip(torch.autograd.grad(y, leaves, gy), torch.autograd.grad(ref, leaves, gy)):
        assert got.shape == want.shape and torch.allclose(got, want, atol=1e-4)
    with torch.no_grad():
        assert torch.equal(blockcopy.linear_act(x, w, b, activation=name, residual=r, dim=dim), y)


@pytest.mark.parametrize("dim,gate,out_norm,in_norm", [(d, g, o, i) for d in (-1, 1) for g in ("none", "channel", "sample") for o, i in
                                                       (("none", "layer"), ("rms", "none"), ("layer", "rms"))])
def test_norm_residual_host_logic(plain_backend, dim, gate, out_norm, in_norm):
    import blockcopy

    gen = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(s, generator=gen).requires_grad_(True)
    shape = (3, 6, 2, 4) if dim == 1 else (3, 2, 4, 6)
    h, y, wo, bo, wi = r(*shape), r(*shape), r(6), r(6), r(6)
    g = {"none": None, "channel": r(6), "sample": r(3, 6, 1, 1) if dim == 1 else r(3, 1, 1, 6)}[gate]
    kw = dict(out_weight=wo, out_bias=bo) if out_norm != "none" else {}
    kw.update(dict(in_weight=wi) if in_norm != "none" else {})
    ho, u = blockcopy.norm_residual(h, y, out_norm=out_norm, gate=g, residual_scale=0.7, in_norm=in_norm, eps=1e-3, dim=dim, **kw)
    last = (lambda t: t.permute(0, 2, 3, 1)) if dim == 1 else (lambda t: t)
    first = (lambda t: t.permute(0, 3, 1, 2)) if dim == 1 else (lambda t: t)
    t = CO.normed(last(y), out_norm, kw.get("out_weight"), kw.get("out_bias"), 1e-3)
    if g is not None:
        t = t * (g if gate == "channel" else last(g))
    h_ref = 0.7 * last(h) + t
    u_ref = None if in_norm == "none" else first(CO.normed(h_ref, in_norm, wi, None, 1e-3))
    h_ref = first(h_ref)
    assert torch.allclose(ho, h_ref, atol=1e-5) and (u is None) == (u_ref is None) and (u is None or torch.allclose(u, u_ref, atol=1e-5))
    outs, refs = [o for o in (ho, u) if o is not None], [o for o in (h_ref, u_ref) if o is not None]
    gs = [torch.randn(o.shape, generator=gen) for o in outs]
    leaves = [h, y] + ([] if g is None else [g]) + list(kw.values())
    for got, want in zip(torch.autograd.grad(outs, leaves, gs), torch.autograd.grad(refs, leaves, gs)):
        assert got.shape == want.shape and torch.allclose(got, want, atol=1e-4)


def test_gradient_of_one_output_only(plain_backend):
    """u alone, or h' alone, may carry the loss; what nobody asked for is not computed; a second derivative is refused."""
    import blockcopy

    h, y = torch.randn(4, 5, requires_grad=True), torch.randn(4, 5)
    for pick in (0, 1):
        out = blockcopy.norm_residual(h, y, in_norm="layer")[pick]
        ref = (h + y) if pick == 0 else CO.normed(h + y, "layer", None, None, 1e-6)
        (a,), (b,) = torch.autograd.grad(out.pow(2).sum(), [h]), torch.autograd.grad(ref.pow(2).sum(), [h])
        assert torch.allclose(a, b, atol=1e-4)
    x, w = torch.randn(3, 4, requires_grad=True), torch.randn(2, 4, requires_grad=True)
    (gx,) = torch.autograd.grad(blockcopy.linear_act(x, w, activation="silu").sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


@pytest.mark.parametrize("shape,dim", [((4, 6), -1), ((2, 3, 6), -1), ((2, 6, 3, 5), 1)])
def test_results_may_be_modified_in_place(plain_backend, shape, dim):
    """As any other operation's results: y.relu_() and its like, with the gradients of the composition."""
    import blockcopy

    gen = torch.Generator().manual_seed(3)
    x, w = torch.randn(shape, generator=gen, requires_grad=True), torch.randn(6, 6, generator=gen, requires_grad=True)
    y = blockcopy.linear_act(x, w, dim=dim)
    h, u = blockcopy.norm_residual(x, y, in_norm="rms", dim=dim)
    got = torch.autograd.grad(h.relu_().sum() + u.mul_(2).pow(2).sum() + blockcopy.linear_act(x, w, dim=dim).add_(1).pow(2).sum(), [x, w])
    rows = x.permute(0, 2, 3, 1) if dim == 1 else x
    yr = rows @ w.t()
    hr, ur = rows + yr, CO.normed(rows + yr, "rms", None, None, 1e-6)
    want = torch.autograd.grad(hr.relu().sum() + (2 * ur).pow(2).sum() + (yr + 1).pow(2).sum(), [x, w])
    assert all(torch.allclose(a, b, atol=1e-3, rtol=1e-4) for a, b in zip(got, want))


def test_no_rows(plain_backend):
    import blockcopy

    x, w = torch.empty(2, 0, 4, requires_grad=True), torch.randn(3, 4, requires_grad=True)
    y = blockcopy.linear_act(x, w, activation="relu")
    assert y.shape == (2, 0, 3)
    gx, gw = torch.autograd.grad(y.sum(), [x, w])
    assert gx.shape == x.shape and torch.equal(gw, torch.zeros_like(w))
    h, v = torch.empty(0, 4, requires_grad=True), torch.ones(4, requires_grad=True)
    ho, u = blockcopy.norm_residual(h, h, in_norm="rms", in_weight=v)
    gh, gv = torch.autograd.grad(ho.sum() + u.sum(), [h, v])
    assert ho.shape == u.shape == gh.shape == (0, 4) and torch.equal(gv, torch.zeros(4))
    h, g = torch.empty(2, 0, 4, requires_grad=True), torch.ones(2, 1, 4, requires_grad=True)
    ho, u = blockcopy.norm_residual(h, h, gate=g)
    gh, gg = torch.autograd.grad(ho.sum(), [h, g])
    assert u is None and ho.shape == gh.shape == (2, 0, 4) and torch.equal(gg, torch.zeros(2, 1, 4))
    for h, g, dim in ((torch.empty(0, 3, 4), torch.ones(0, 1, 4), -1), (torch.empty(0, 4, 2, 2), torch.ones(0, 4, 1, 1), 1)):        # no samples: no gates either
        h.requires_grad_(True), g.requires_grad_(True)
        ho, u = blockcopy.norm_residual(h, h, gate=g, in_norm="layer", dim=dim)
        gh, gg = torch.autograd.grad(ho.sum() + u.sum(), [h, g])
        assert ho.shape == u.shape == gh.shape == h.shape and gg.shape == g.shape


# ------------------------------------------------------------------------------------------------ GPU
def _rand(gen, *shape, dtype=torch.float32, std=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * std + mean).to(dtype).cuda()


def _linear_case(dt, M, K, N, name, bias=True, res=False, train=False, bias_dtype=None, seed=0, pad=0):
    """pad: extra elements between rows, so that row strides differ from the widths."""
    import blockcopy

    gen = torch.Generator().manual_seed(seed)
    dtype = DT[dt]
    wide = lambda r, c, std=1.0: _rand(gen, r, c + pad, dtype=dtype, std=std)[:, pad // 2:pad // 2 + c]
    x, w = wide(M, K), wide(N, K, K ** -0.5)
    b = _rand(gen, N, dtype=bias_dtype or dtype, std=0.3) if bias else None
    r = wide(M, N) if res else None
    gy = wide(M, N) if train else None
    leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None] if train else []
    y = blockcopy.linear_act(x, w, b, activation=name, residual=r)
    want = CO.linear(x.detach(), w.detach(), None if b is None else b.detach(), None if r is None else r.detach(), name, gy)
    _close(y.detach(), *want["y"], (dt, M, K, N, name, "y"))
    if train:
        got = dict(zip([n for n, t in (("dx", x), ("dw", w), ("db", b), ("dr", r)) if t is not None], torch.autograd.grad(y, leaves, gy)))
        for k in ("dx", "dw", "db"):
            if k in got:
                _close(got[k], *want[k], (dt, M, K, N, name, k))
        if r is not None:
            assert torch.equal(got["dr"], gy)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("M,K,N", [(1, 16, 16), (1, 515, 1001), (1, 2048, 24), (2, 1, 1), (5, 64, 64), (13, 129, 33), (16, 256, 512), (17, 1000, 7), (33, 96, 130), (63, 320, 65),
                                   (64, 513, 200), (65, 72, 129), (127, 1, 256), (128, 128, 128), (200, 65, 64), (257, 264, 300), (300, 31, 31), (1000, 64, 19)])
def test_linear_forward(dt, M, K, N):
    """Sizes around every tile edge, odd ones, one row; alternately with bias, residual, activation."""
    i = M + K + N
    _linear_case(dt, M, K, N, CO.ACTS[i % 5], bias=i % 2 == 0, res=i % 3 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("name", CO.ACTS)
def test_linear_activations_and_gradients(dt, name):
    _linear_case(dt, 130, 96, 72, name, bias=True, res=True, train=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("M,K,N", [(1, 32, 48), (1, 1, 1), (3, 17, 1000), (31, 515, 9), (129, 33, 257), (513, 64, 64), (1027, 24, 40), (2049, 19, 130), (4100, 128, 8)])
def test_linear_gradients(dt, M, K, N):
    """Long and short sums in every product; odd sizes; one row."""
    _linear_case(dt, M, K, N, ("silu", "none", "gelu")[(M + N) % 3], bias=True, train=True, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("pad", [1, 6, 16])
def test_linear_row_strides(dt, pad):
    """Rows of a wider matrix: odd starts, strides with and without vectors."""
    _linear_case(dt, 70, 64, 72, "gelu", res=True, train=True, pad=pad, seed=5)
    _linear_case(dt, 3, 136, 40, "none", res=True, pad=pad, seed=6)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
def test_linear_large_odd_rows_of_wider_matrices(dt):
    """Operands that are brought into order first: odd widths, rows of a wider matrix, with and without an activation."""
    _linear_case(dt, 1100, 1003, 1001, "silu", train=True, pad=3, seed=8)
    _linear_case(dt, 1100, 1001, 1001, "none", train=True, pad=8, seed=9)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_linear_bias_in_float32(dt):
    _linear_case(dt, 40, 48, 56, "gelu", train=True, bias_dtype=torch.float32, seed=7)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("M,K,N", [(1, 1024, 260), (9, 1023, 65), (40, 640, 96), (300, 512, 384), (260, 1000, 270), (2500, 40, 96)])
def test_linear_whole_numbers_are_exact(dt, M, K, N):
    """Small whole numbers: every partial sum is exact in float32, so outputs are the correctly rounded results, all of them."""
    import blockcopy

    gen = torch.Generator().manual_seed(11)
    pick = lambda *s: torch.randint(-3, 4, s, generator=gen).to(DT[dt]).cuda()
    x, w, b, r = pick(M, K).requires_grad_(True), pick(N, K).requires_grad_(True), pick(N).requires_grad_(True), pick(M, N)
    y = blockcopy.linear_act(x, w, b, residual=r)
    d = lambda t: t.detach().double()
    assert torch.equal(y, (d(x) @ d(w).t() + d(b) + d(r)).to(DT[dt]))
    gy = pick(M, N)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], gy)
    assert torch.equal(gx, (d(gy) @ d(w)).to(DT[dt])) and torch.equal(gw, (d(gy).t() @ d(x)).to(DT[dt])) and torch.equal(gb, d(gy).sum(0).to(DT[dt]))
    # relu's gradient: zero and below pass nothing
    y = blockcopy.linear_act(x, w, b, activation="relu")
    z = d(x) @ d(w).t() + d(b)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], gy)
    dz = d(gy) * (z > 0)
    assert torch.equal(gx, (dz @ d(w)).to(DT[dt])) and torch.equal(gw, (dz.t() @ d(x)).to(DT[dt])) and torch.equal(gb, dz.sum(0).to(DT[dt]))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("M,K,N", [(4100, 72, 4104), (4104, 4104, 72), (72, 4104, 4104), (4099, 136, 4101), (8200, 1032, 2056), (8192, 576, 2048), (2100, 1001, 1003), (1500, 1002, 1004)])
def test_linear_large_tiles_are_exact(dt, M, K, N):
    """Enough work for the large tile in each of the three products (and, with odd sizes, what takes its place): whole numbers, exact results."""
    import blockcopy

    gen = torch.Generator(device="cuda").manual_seed(12)
    pick = lambda *s: torch.randint(-2, 3, s, generator=gen, device="cuda").to(DT[dt])
    x, w, b, gy = pick(M, K).requires_grad_(True), pick(N, K).requires_grad_(True), pick(N).requires_grad_(True), pick(M, N)
    y = blockcopy.linear_act(x, w, b, activation="relu")
    d = lambda t: t.detach().double()
    z = d(x) @ d(w).t() + d(b)
    assert torch.equal(y, z.clamp_min(0).to(DT[dt]))
    dz = d(gy) * (z > 0)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], gy)
    assert torch.equal(gx, (dz @ d(w)).to(DT[dt])) and torch.equal(gw, (dz.t() @ d(x)).to(DT[dt])) and torch.equal(gb, dz.sum(0).to(DT[dt]))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("M,K,N", [(2048, 1024, 2048), (2040, 1000, 2024), (3000, 768, 2304), (4000, 600, 4000), (4000, 4000, 600), (600, 4000, 4000), (4099, 33, 4101), (4099, 4101, 33),
                                   (33, 4101, 4099), (512, 4096, 1000), (100, 1032, 4096), (16384, 136, 264)])
def test_linear_every_tile_is_exact(dt, M, K, N):
    """Every tile, wave and slice shape (partial tiles and steps among them) in each product it is used for."""
    test_linear_large_tiles_are_exact(dt, M, K, N)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("M", [1, 20, 300])
def test_linear_infinities_stay_in_their_rows(dt, M):
    """An infinity or NaN in a row of x reaches that row's outputs only, one in a row of w that column's; large finite pre-activations keep
    every activation's gradient finite."""
    import blockcopy

    gen = torch.Generator().manual_seed(13)
    x, w = _rand(gen, M, 70, dtype=DT[dt]), _rand(gen, 50, 70, dtype=DT[dt])
    clean = blockcopy.linear_act(x, w)
    xb, wb = x.clone(), w.clone()
    xb[M // 2, 69] = float("inf")
    wb[49, 0] = float("nan")
    y = blockcopy.linear_act(xb, wb)
    keep = torch.ones_like(clean, dtype=torch.bool)
    keep[M // 2], keep[:, 49] = False, False
    assert torch.equal(y[keep], clean[keep]) and bool(y[:, 49].isnan().all()) and bool(torch.isinf(y[M // 2, :49]).all())
    big = (w.abs() + 0.5).requires_grad_(True)
    for name, sign in itertools.product(CO.ACTS, (1.0, -1.0)):
        xs = torch.full_like(x, sign * 100.0).requires_grad_(True)
        y = blockcopy.linear_act(xs, big, activation=name)
        for t in (y, *torch.autograd.grad(y, [xs, big], torch.ones_like(y))):
            assert bool(t.isfinite().all()), (name, sign)


NORM_SIZES = [(1, 1), (1, 16), (3, 7), (5, 8), (70, 24), (33, 64), (9, 100), (20, 255), (6, 256), (130, 512), (7, 513), (12, 1000), (5, 1024), (4, 1999), (3, 2048), (3, 4096), (2, 4100),
              (2, 8192), (3, 8193), (2, 12000), (1, 16384)]


def _norm_case(dt, M, C, out_norm, in_norm, gate="channel", scale=1.0, bias=True, groups=1, block=True, pf32=False, train=True, pad=0, seed=0, eps=1e-6, mean=0.3, weights=True):
    import blockcopy

    gen = torch.Generator().manual_seed(seed)
    dtype = DT[dt]
    pd = torch.float32 if pf32 else dtype
    rpg = M // groups if gate == "sample" else 0
    wide = lambda std, m=0.0: _rand(gen, M, C + pad, dtype=dtype, std=std, mean=m)[:, pad // 2:pad // 2 + C]
    h, y = wide(1.5, mean), wide(0.8, mean) if block else None
    vec = lambda on, std, m: _rand(gen, C, dtype=pd, std=std, mean=m) if on else None
    p = {"wo": vec(weights and out_norm != "none", 0.3, 1.0), "bo": vec(bias and out_norm != "none", 0.2, 0.0), "wi": vec(weights and in_norm != "none", 0.3, 1.0),
         "bi": vec(bias and in_norm != "none", 0.2, 0.0)}
    g = None if gate == "none" or not block else _rand(gen, *((groups, C) if rpg else (C,)), dtype=pd, std=0.3, mean=0.6)
    names = [n for n, t in (("h", h), ("y", y), ("wo", p["wo"]), ("bo", p["bo"]), ("gate", g), ("wi", p["wi"]), ("bi", p["bi"])) if t is not None]
    leaves = [{"h": h, "y": y, "gate": g, **p}[n] for n in names]
    if train:
        [t.requires_grad_(True) for t in leaves]
    hv = h.view(groups, rpg, C) if rpg and pad == 0 else h
    yv = y.view(groups, rpg, C) if rpg and pad == 0 and block else y
    gv = g.view(groups, 1, C) if rpg and pad == 0 else g
    ho, u = blockcopy.norm_residual(hv, yv, out_norm=out_norm, out_weight=p["wo"], out_bias=p["bo"], gate=gv, residual_scale=scale, in_norm=in_norm, in_weight=p["wi"],
                                    in_bias=p["bi"], eps=eps)
    # the definition and its gradients in 64 bits
    dd = {n: t.detach().cpu().double().requires_grad_(True) for n, t in zip(names, leaves)}
    rh, ru = CO.norm_residual(dd["h"], dd.get("y"), {k: dd.get(k) for k in p}, dd.get("gate"), scale, out_norm, in_norm, eps, rpg)
    a = {n: t.detach().abs() for n, t in dd.items()}
    U = CO.U
    one = torch.ones(1, dtype=torch.float64)
    # every statistic is a tree of at most 64 float32 roundings; what it normalises keeps the size of its row's mean besides its own
    def norm_err(x, dx, kind, w, b):
        x, dx = x.detach(), dx
        if kind == "none":
            return x.abs(), dx, one * 0, x * 0
        m = x.mean(-1, keepdim=True) if kind == "layer" else x * 0
        c = x - m
        rs = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
        n = c * rs
        d = dx + 64 * U * (x.abs() + x.abs().mean(-1, keepdim=True) * (kind == "layer"))       # error of the centred value
        d = d + (d.mean(-1, keepdim=True) if kind == "layer" else 0)
        ne = rs * d + n.abs() * (rs * rs * (c.abs() * d).mean(-1, keepdim=True) + 64 * U)          # ... of the normalised one
        w = one if w is None else w
        return n.abs() * w + (0 if b is None else b), ne * w + 4 * U * (n.abs() * w + (0 if b is None else b)), ne, rs
    h_err = torch.zeros(M, C, dtype=torch.float64)
    nyn = ny_err = None
    gfull = one if g is None else (a["gate"].repeat_interleave(rpg, 0) if rpg else a["gate"])
    if block:
        ta, te, ny_err, rsy = norm_err(dd["y"], torch.zeros(M, C, dtype=torch.float64), out_norm, a.get("wo"), a.get("bo"))
        h_err = gfull * te + 4 * U * (gfull * ta + scale * a["h"])
        _close(ho.detach().reshape(M, C), rh.detach(), CO.rounded(rh.detach(), h_err, dtype), (dt, M, C, "h"))
    else:
        assert ho is hv
    if in_norm != "none":
        ua, ue, nh_err, rsh = norm_err(rh, h_err, in_norm, a.get("wi"), a.get("bi"))
        _close(u.detach().reshape(M, C), ru.detach(), CO.rounded(ru.detach(), ue, dtype), (dt, M, C, "u"))
    if not train:
        return
    gh, gu = wide(1.0) if block else None, wide(1.0) if in_norm != "none" else None
    outs = [(o, r, q) for o, r, q in ((ho if block else None, rh if block else None, gh), (u, ru, gu)) if q is not None]
    got = dict(zip(names, torch.autograd.grad([o for o, _, _ in outs], leaves, [q.reshape(o.shape) for o, _, q in outs])))
    ref = dict(zip(names, torch.autograd.grad([r for _, r, _ in outs], [dd[n] for n in names], [q.cpu().double() for _, _, q in outs])))
    # bounds: sizes of all terms of a gradient, times its 128 roundings, plus the errors of the normalised rows it contains
    def bwd_err(p_, pe, n, ne, rs, kind):
        """error of rs (p - mean p - n mean(p n)) given errors of p and n"""
        mp, mn = (p_ * n).mean(-1, keepdim=True), (pe * n + p_ * ne).mean(-1, keepdim=True)
        lay = kind == "layer"
        size = rs * (p_ + lay * p_.mean(-1, keepdim=True) + n * mp)
        rel = 64 * U + (ne * n).mean(-1, keepdim=True)
        return rs * (pe + lay * pe.mean(-1, keepdim=True) + n * mn + ne * mp) + (128 * U + rel) * size, size
    gcur, gerr = (gh.cpu().double().abs() if block else one * 0), torch.zeros(M, C, dtype=torch.float64)
    bounds = {}
    if in_norm != "none":
        x = rh.detach()
        c = x - (x.mean(-1, keepdim=True) if in_norm == "layer" else 0)
        n = (c * rsh).abs()
        q = gu.cpu().double().abs()
        wi = a.get("wi", one)
        bounds["wi"] = ((q * nh_err) + (M + 4) * U * q * n).sum(0) + M * U * (q * n).sum(0)
        bounds["bi"] = (M + 1) * U * q.sum(0)
        e, size = bwd_err(q * wi, 2 * U * q * wi, n, nh_err, rsh, in_norm)
        gerr, gcur = gerr + e + 2 * U * (gcur + size), gcur + size
    bounds["h"] = abs(scale) * (gerr + 2 * U * gcur)
    if block:
        if out_norm != "none":
            x = dd["y"].detach()
            c = x - (x.mean(-1, keepdim=True) if out_norm == "layer" else 0)
            n = (c * rsy).abs()
        else:
            n, ny_err = a["y"], torch.zeros(M, C, dtype=torch.float64)
        rows = lambda t: t.view(groups, rpg, C).sum(1) if rpg else t.sum(0)
        bounds["gate"] = rows(gerr * ta + gcur * te) + 2 * (M + 4) * U * rows(gcur * ta)
        q, qe = gcur * gfull, gerr * gfull + 2 * U * gcur * gfull
        bounds["wo"] = (qe * n + q * ny_err).sum(0) + 2 * (M + 4) * U * (q * n).sum(0)
        bounds["bo"] = qe.sum(0) + 2 * (M + 4) * U * q.sum(0)
        wo = a.get("wo", one)
        bounds["y"] = bwd_err(q * wo, qe * wo + 2 * U * q * wo, n, ny_err, rsy, out_norm)[0] if out_norm != "none" else qe
    for k, v in ref.items():
        _close(got[k], v, CO.rounded(v, bounds[k], dtype if k in ("h", "y") else pd), (dt, M, C, out_norm, in_norm, gate, "d" + k))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("M,C", NORM_SIZES)
def test_norm_sizes(dt, M, C):
    i = M + C
    _norm_case(dt, M, C, ("rms", "layer")[i % 2] if C > 1 else "rms", ("layer", "rms")[i % 3 % 2] if C > 1 else "rms", seed=i)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("out_norm,in_norm", list(itertools.product(("none", "rms", "layer"), repeat=2)))
def test_norm_kinds(dt, out_norm, in_norm):
    _norm_case(dt, 37, 96, out_norm, in_norm, gate="none", scale=0.7, seed=1)
    _norm_case(dt, 37, 96, out_norm, in_norm, gate="channel", bias=False, seed=2)
    _norm_case(dt, 36, 72, out_norm, in_norm, gate="sample", groups=9, seed=3)
    _norm_case(dt, 5, 40, out_norm, in_norm, gate="channel", weights=False, bias=False, seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
def test_norm_without_a_block_and_many_rows(dt):
    _norm_case(dt, 50, 120, "none", "layer", block=False, gate="none", seed=5)
    _norm_case(dt, 1, 300, "none", "rms", block=False, gate="none", seed=6)
    _norm_case(dt, 9001, 16, "rms", "layer", seed=7)
    _norm_case(dt, 4200, 48, "layer", "rms", gate="sample", groups=2100, seed=8)
    _norm_case(dt, 130, 8200, "layer", "none", seed=13)
    _norm_case(dt, 130, 9001, "none", "layer", block=False, gate="none", seed=14)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_norm_float32_parameters(dt):
    _norm_case(dt, 40, 200, "layer", "rms", pf32=True, seed=9)
    _norm_case(dt, 30, 77, "rms", "layer", pf32=True, gate="sample", groups=3, seed=10)
    _norm_case(dt, 12, 9000, "rms", "layer", pf32=True, gate="sample", groups=3, seed=12)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("pad", [1, 8])
def test_norm_row_strides(dt, pad):
    _norm_case(dt, 21, 200, "layer", "rms", pad=pad, seed=11)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
def test_norm_rows_are_independent(dt):
    """A row of zeros gives zeros (eps keeps it finite), an infinity or NaN stays in its row."""
    import blockcopy

    gen = torch.Generator().manual_seed(17)
    h, y = _rand(gen, 40, 136, dtype=DT[dt]), _rand(gen, 40, 136, dtype=DT[dt])
    kw = dict(out_norm="layer", in_norm="rms")
    h0, u0 = blockcopy.norm_residual(h, y, **kw)
    h, y = h.clone(), y.clone()
    h[3], y[3], h[17, 135], y[30, 0] = 0, 0, float("inf"), float("nan")
    h1, u1 = blockcopy.norm_residual(h, y, **kw)
    keep = torch.ones(40, dtype=torch.bool)
    keep[[3, 17, 30]] = False
    assert torch.equal(h1[keep], h0[keep]) and torch.equal(u1[keep], u0[keep])
    assert not bool(h1[3].any()) and not bool(u1[3].any()) and bool(u1[17, 135].isnan()) and bool(h1[30].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("M,K,N", [(70, 40, 24), (1100, 1026, 1030)])
def test_each_linear_gradient_alone(dt, M, K, N):
    """Frozen arguments (a bias tuned alone, a first layer's input) change no bit of the other gradients."""
    import blockcopy

    gen = torch.Generator().manual_seed(47)
    ts = [_rand(gen, M, K, dtype=DT[dt]), _rand(gen, N, K, dtype=DT[dt], std=K ** -0.5), _rand(gen, N, dtype=DT[dt]), _rand(gen, M, N, dtype=DT[dt])]
    gy = _rand(gen, M, N, dtype=DT[dt])
    for act in ("none", "gelu"):
        def grads(live):
            args = [t.clone().requires_grad_(i in live) for i, t in enumerate(ts)]
            return torch.autograd.grad(blockcopy.linear_act(args[0], args[1], args[2], act, args[3]), [args[i] for i in live], gy)

        full = grads(range(4))
        for live in itertools.chain(*(itertools.combinations(range(4), r) for r in (1, 2, 3))):
            assert all(torch.equal(g, full[i]) for i, g in zip(live, grads(live))), (act, live)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("C", [40, 1030, 9000])
def test_each_norm_gradient_alone(dt, C):
    import blockcopy

    gen = torch.Generator().manual_seed(53)
    M = 60
    ts = [_rand(gen, M, C, dtype=DT[dt]), _rand(gen, M, C, dtype=DT[dt]), *(_rand(gen, C, dtype=DT[dt], mean=1.0, std=0.2) for _ in range(5))]
    gs = [_rand(gen, M, C, dtype=DT[dt]) for _ in range(2)]

    def grads(live, use):
        a = [t.clone().requires_grad_(i in live) for i, t in enumerate(ts)]
        out = blockcopy.norm_residual(a[0], a[1], out_norm="layer", out_weight=a[2], out_bias=a[3], gate=a[4], in_norm="rms", in_weight=a[5], in_bias=a[6])
        return torch.autograd.grad([out[i] for i in use], [a[i] for i in live], [gs[i] for i in use])

    for use in ((0, 1), (1,)):
        full = grads(range(7), use)
        for i in range(7):
            assert torch.equal(grads([i], use)[0], full[i]), (use, i)


@pytest.mark.gpu
def test_results_repeat_bit_for_bit():
    import blockcopy

    gen = torch.Generator().manual_seed(19)
    x, w, gy = _rand(gen, 3000, 200, dtype=torch.bfloat16).requires_grad_(True), _rand(gen, 96, 200, dtype=torch.bfloat16).requires_grad_(True), _rand(gen, 3000, 96, dtype=torch.bfloat16)
    v = _rand(gen, 96, dtype=torch.bfloat16).requires_grad_(True)

    def once():
        y = blockcopy.linear_act(x, w, v, activation="gelu")
        h, u = blockcopy.norm_residual(gy, y, out_norm="layer", out_weight=v, gate=v, in_norm="rms", in_weight=v)
        return [h, u, *torch.autograd.grad((h, u), [x, w, v], (gy, gy))]

    a, b = once(), once()
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def _block(x, ps, dim=-1):
    """Two residual blocks as a user writes them: norm -> widen -> narrow -> norm, gate, residual, next norm."""
    import blockcopy

    h, u = blockcopy.norm_residual(x, in_norm="layer", in_weight=ps["n0"], dim=dim)
    for i in (1, 2):
        y = blockcopy.linear_act(u, ps[f"a{i}"], ps[f"ab{i}"], activation="gelu", dim=dim)
        y = blockcopy.linear_act(y, ps[f"b{i}"], ps[f"bb{i}"], dim=dim)
        h, u = blockcopy.norm_residual(h, y, out_norm="rms", out_weight=ps[f"o{i}"], gate=ps[f"g{i}"], in_norm="layer", in_weight=ps[f"n{i}"], dim=dim)
    return blockcopy.linear_act(u, ps["b1"].t().contiguous() if dim == -1 else ps["b1"].t().contiguous(), residual=None, dim=dim), h


def _block_ref(x, ps):
    u = CO.normed(x, "layer", ps["n0"], None, 1e-6)
    h = x
    for i in (1, 2):
        y = CO.act(u @ ps[f"a{i}"].t() + ps[f"ab{i}"], "gelu")[0] @ ps[f"b{i}"].t() + ps[f"bb{i}"]
        h = h + ps[f"g{i}"] * CO.normed(y, "rms", ps[f"o{i}"], None, 1e-6)
        u = CO.normed(h, "layer", ps[f"n{i}"], None, 1e-6)
    return u @ ps["b1"], h


def _block_params(C, dtype, seed=23):
    gen = torch.Generator().manual_seed(seed)
    ps = {"n0": _rand(gen, C, dtype=dtype, std=0.1, mean=1.0)}
    for i in (1, 2):
        ps.update({f"a{i}": _rand(gen, 2 * C, C, dtype=dtype, std=C ** -0.5), f"ab{i}": _rand(gen, 2 * C, dtype=dtype, std=0.1), f"b{i}": _rand(gen, C, 2 * C, dtype=dtype, std=(2 * C) ** -0.5),
                   f"bb{i}": _rand(gen, C, dtype=dtype, std=0.1), f"o{i}": _rand(gen, C, dtype=dtype, std=0.1, mean=1.0), f"g{i}": _rand(gen, C, dtype=dtype, std=0.1, mean=0.5),
                   f"n{i}": _rand(gen, C, dtype=dtype, std=0.1, mean=1.0)})
    return ps


@pytest.mark.gpu
def test_run_of_blocks_and_its_gradients():
    """A run of both operators, forward and backward, against the 64-bit composition (float32: about 20 operations deep, each within a few
    hundred roundings of its values, all of order one: 2e-4 of the largest element covers their sum many times over)."""
    ps = {k: v.requires_grad_(True) for k, v in _block_params(72, torch.float32).items()}
    gen = torch.Generator().manual_seed(29)
    x = _rand(gen, 3, 50, 72).requires_grad_(True)
    outs = _block(x, ps)
    d = {k: v.detach().double().requires_grad_(True) for k, v in ps.items()}
    xd = x.detach().double().requires_grad_(True)
    refs = _block_ref(xd, d)
    gs = [_rand(gen, *o.shape) for o in outs]
    got = torch.autograd.grad(outs, [x, *ps.values()], gs, allow_unused=True)
    want = torch.autograd.grad(refs, [xd, *d.values()], [g.double() for g in gs], allow_unused=True)
    for a, b in zip((*outs, *got), (*refs, *want)):
        assert (a is None) == (b is None)
        if a is not None:
            assert float((a.double() - b).abs().max()) <= 2e-4 * float(b.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DT)
def test_packed_tiles_give_what_dense_maps_give(dt):
    """On packed tiles (TensorWrapper) the operators give the executed tiles of the dense map's result, bit for bit; skipped tiles keep the
    previous frame's values when the result is combined."""
    import blockcopy
    from blockcopy.core.blockcopy import BlockCopyModel  # noqa: F401  (the wrapper's own import path)

    C, bs = 72, 8
    ps = _block_params(C, DT[dt])
    gen = torch.Generator().manual_seed(31)
    frames = [_rand(gen, 1, C, 24, 32, dtype=DT[dt]).contiguous(memory_format=torch.channels_last) for _ in range(2)]
    grids = [torch.ones(1, 1, 3, 4, dtype=torch.bool), torch.rand(1, 1, 3, 4, generator=gen) < 0.5]
    prev, last = None, None
    for x, grid in zip(frames, grids):
        dense = _block(x, ps, dim=1)[1]
        t = blockcopy.to_tensorwrapper(x)
        feats = t.process_temporal_features(prev)
        out = _block(t.to_blocks(grid.cuda(), grid), ps)[1]
        assert blockcopy.is_block(out)
        got = out.combine().to_tensor()
        mask = grid.repeat_interleave(bs, 2).repeat_interleave(bs, 3).cuda()
        want = dense if last is None else torch.where(mask, dense, last)
        assert torch.equal(got, want)
        prev, last = feats, got.clone()


@pytest.mark.gpu
def test_captured_and_replayed():
    """Forward and backward in one graph, two graphs side by side, replays on changed inputs, against eager runs."""
    import blockcopy

    gen = torch.Generator().manual_seed(37)
    mk = lambda *s: _rand(gen, *s, dtype=torch.float16)
    ins = [[mk(513, 1000), mk(40, 1000), mk(40), mk(513, 40)] for _ in range(3)]
    side, streams = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    graphs = []
    for _ in range(2):
        live = [t.clone().requires_grad_(i < 3) for i, t in enumerate(ins[0])]

        def step(live=live):
            y = blockcopy.linear_act(live[0], live[1], live[2], activation="gelu")
            h, u = blockcopy.norm_residual(live[3], y, out_norm="rms", gate=live[2], in_norm="layer")
            return [h.detach(), u.detach(), *torch.autograd.grad((h, u), live[:3], (live[3], live[3]))]

        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs = step()
        graphs.append((g, live, outs, step))
    for r in range(4):
        for k, (g, live, outs, step) in enumerate(graphs):
            with torch.no_grad():
                for a, b in zip(live, ins[(r + k) % 3]):
                    a.copy_(b)
        torch.cuda.synchronize()
        for (g, *_), s in zip(graphs, streams):        # (at once, each on a stream of its own)
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        want = []
        for k in range(2):
            x, w, b, s = [t.clone() for t in ins[(r + k) % 3]]
            [t.requires_grad_(True) for t in (x, w, b)]
            y = blockcopy.linear_act(x, w, b, activation="gelu")
            h, u = blockcopy.norm_residual(s, y, out_norm="rms", gate=b, in_norm="layer")
            want.append([h.detach(), u.detach(), *torch.autograd.grad((h, u), [x, w, b], (s, s))])
            del h, u, y
        for k in range(2):
            for i, (a, b) in enumerate(zip(graphs[k][2], want[k])):
                assert torch.equal(a, b), (r, k, i)


@pytest.mark.gpu
def test_on_another_stream_and_two_at_once():
    """Calls on two streams at a time own their workspaces."""
    import blockcopy

    gen = torch.Generator().manual_seed(41)
    x, w = _rand(gen, 20, 8000, dtype=torch.bfloat16), _rand(gen, 130, 8000, dtype=torch.bfloat16)
    want = blockcopy.linear_act(x, w, activation="silu")
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(blockcopy.linear_act(x, w, activation="silu"))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for g in got for t in g)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 20])
def test_very_many_columns(M):
    """One launch of the kernel for few rows has fewer than 2^32 threads: beyond its columns the tiles take over."""
    import blockcopy

    N = 70_000_003 if M == 1 else 9_000_001
    w = (torch.arange(N, device="cuda") % 1021).to(torch.float16)[:, None]
    x = torch.arange(1, M + 1, device="cuda", dtype=torch.float16)[:, None]
    y = blockcopy.linear_act(x, w)
    for m in {0, M - 1}:        # (whole numbers: exact up to 2048, rounded once beyond)
        assert torch.equal(y[m], (w[:, 0].float() * (m + 1)).half())


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements in one operand: rows at the far end are read and written at their own places."""
    import blockcopy

    M, K = (1 << 31) // 512 + 300, 512
    x = torch.zeros((M, K), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(43)
    x[-300:] = _rand(gen, 300, K, dtype=torch.bfloat16)
    w = _rand(gen, 24, K, dtype=torch.bfloat16)
    y = blockcopy.linear_act(x, w)
    # (not bit for bit against a call on the far rows alone: how a long sum is split goes by the number of rows)
    _close(y[-300:], *CO.linear(x[-300:], w, None, None, "none")["y"], "far rows")
    assert not bool(y[:-300].any())
    del y
    h, u = blockcopy.norm_residual(x, x, in_norm="rms")
    h2, u2 = blockcopy.norm_residual(x[-300:].clone(), x[-300:].clone(), in_norm="rms")
    assert torch.equal(h[-300:], h2) and torch.equal(u[-300:], u2) and not bool(u[:1000].any())

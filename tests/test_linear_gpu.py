"""cudair_linear, cudair_gated and their gradients against their definitions in
64 bits (linear_ref.py derives the tolerances): sizes from one row to several
tiles, odd and ragged ones, both weight layouts, both 16-bit types, fp32
outputs, pitches and alignments, empty sizes, and the four as one layer."""
import pytest

from linear_ref import (Out, act64, act_error, act_grad64, grad_error, half_ulp, normal, padded, sum_error)

pytestmark = pytest.mark.gpu

# M, N, K: single rows, both sides of 16, 64 and 128 rows, tile edges, odd sizes.
SHAPES = [(1, 1, 1), (1, 8, 64), (1, 1000, 4096), (2, 131, 70), (7, 515, 1024), (16, 256, 512), (17, 300, 77),
          (33, 1024, 200), (64, 129, 2048), (65, 640, 333), (100, 96, 64), (128, 384, 1000), (129, 257, 65),
          (200, 72, 4096), (256, 256, 64), (257, 1031, 519), (400, 2050, 136), (1025, 513, 96),
          (257, 5000, 200), (1290, 1031, 1100), (600, 2050, 5000)]  # enough tiles for the persistent pairs
FORMS = [  # dtype, rows, act, bias, residual, z, fp32 output, pitch padding, lead
    ("bf16", True, "none", None, True, False, False, 8, 0),
    ("fp16", False, "gelu_tanh", "f32", False, True, False, 0, 8),
    ("bf16", False, "silu", "16", True, True, True, 8, 8),
    ("fp16", True, "gelu", "16", True, False, False, 24, 0),
    ("bf16", True, "relu", "f32", False, True, False, 0, 0),
]


def _dt(name):
    import torch
    return torch.bfloat16 if name == "bf16" else torch.float16


def _gen(dev, *key):
    import torch
    g = torch.Generator(device=dev)
    g.manual_seed(hash(key) % (1 << 31))
    return g


def _weight(g, N, K, dt, dev, rows, pad=8, lead=0):
    std = max(K, 1) ** -0.5
    return normal(g, N, K, dt, dev, std, pad, lead) if rows else normal(g, K, N, dt, dev, std, pad, lead)


def _kn(w, rows):
    """The weight as a K x N matrix in 64 bits."""
    return w.double().t() if rows else w.double()


@pytest.mark.parametrize("form", FORMS, ids=lambda f: "-".join(str(x) for x in f))
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(dev, cudair, M, N, K, form):
    import torch
    from cudair import kernels
    dtype, rows, act, bias, residual, z, f32, pad, lead = form
    dt = _dt(dtype)
    dd = torch.float32 if f32 else dt
    g = _gen(dev, M, N, K)
    a = normal(g, M, K, dt, dev, 1.0, pad, lead)
    b = _weight(g, N, K, dt, dev, rows, pad, lead)
    bv = None if bias is None else torch.randn(N, generator=g, device=dev).to(torch.float32 if bias == "f32" else dt)
    r = normal(g, M, N, dd, dev, 1.0, pad, lead) if residual else None
    d, zo = Out(M, N, dd, dev, pad, lead), Out(M, N, dt, dev, pad, lead) if z else None
    kernels.linear(a, b, d.t, bias=bv, residual=r, z=zo.t if z else None, act=act, b_trans=rows)
    torch.cuda.synchronize()
    A, B = a.double(), _kn(b, rows)
    Z = A @ B + (0 if bv is None else bv.double())
    dz = sum_error(A.abs() @ B.abs() + (0 if bv is None else bv.double().abs()), K)
    D = act64(Z, act) + (r.double() if residual else 0)
    extra = (act64(Z, act).abs() + D.abs()) * 2.0 ** -23  # the residual's fp32 add
    d.check("d", D, half_ulp(D, dd) + act_error(Z, dz, act) + extra)
    if z:
        zo.check("z", Z, half_ulp(Z, dt) + dz)
    assert kernels.wait_status(clear=True) == 0


@pytest.mark.parametrize("dtype,rows,act,save,pad,lead", [("bf16", True, "silu", True, 8, 0),
                                                          ("fp16", False, "gelu_tanh", False, 0, 8),
                                                          ("bf16", False, "gelu", True, 24, 8),
                                                          ("fp16", True, "relu", False, 0, 0),
                                                          ("bf16", True, "none", True, 8, 8)])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gated(dev, cudair, M, N, K, dtype, rows, act, save, pad, lead):
    import torch
    from cudair import kernels
    dt = _dt(dtype)
    g = _gen(dev, M, N, K, 1)
    x = normal(g, M, K, dt, dev, 1.0, pad, lead)
    wg, wu = (_weight(g, N, K, dt, dev, rows, pad, lead) for _ in range(2))
    h, go, uo = (Out(M, N, dt, dev, pad, lead) for _ in range(3))
    kernels.gated(x, wg, wu, h.t, g=go.t if save else None, u=uo.t if save else None, act=act, b_trans=rows)
    torch.cuda.synchronize()
    X, G, U = x.double(), _kn(wg, rows), _kn(wu, rows)
    eg, eu = sum_error(X.abs() @ G.abs(), K), sum_error(X.abs() @ U.abs(), K)
    G, U = X @ G, X @ U
    H = act64(G, act) * U
    ea = act_error(G, eg, act)
    h.check("h", H, half_ulp(H, dt) + ea * (U.abs() + eu) + act64(G, act).abs() * eu + H.abs() * 2.0 ** -23)
    if save:
        go.check("g", G, half_ulp(G, dt) + eg)
        uo.check("u", U, half_ulp(U, dt) + eu)
    assert kernels.wait_status(clear=True) == 0


def _check_product(name, out, P, Q, dP, dQ, K, dt, more=None):
    """out = P @ Q, where an operand may be off by dP, dQ (its rounding)."""
    ref, mag = P @ Q, P.abs() @ Q.abs()
    err = sum_error(mag, K)
    if dP is not None:
        err = err + dP @ Q.abs()
    if dQ is not None:
        err = err + P.abs() @ dQ
    if more is not None:
        ref, err = ref + more[0], err + more[1]
    out.check(name, ref, half_ulp(ref, dt) + err)
    return ref, err


@pytest.mark.parametrize("dtype,rows,act,dy32,da32,db32,inplace", [
    ("bf16", True, "gelu_tanh", False, False, False, None), ("fp16", False, "silu", True, True, False, None),
    ("bf16", False, "relu", False, False, True, "z"), ("fp16", True, "gelu", False, True, True, "dy"),
    ("bf16", True, "none", False, False, False, None), ("bf16", False, "none", True, True, True, None)])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_backward(dev, cudair, M, N, K, dtype, rows, act, dy32, da32, db32, inplace):
    import torch
    from cudair import kernels
    dt, f32 = _dt(dtype), torch.float32
    g = _gen(dev, M, N, K, 2)
    a, b = normal(g, M, K, dt, dev), _weight(g, N, K, dt, dev, rows)
    dy = normal(g, M, N, f32 if dy32 else dt, dev)
    z = normal(g, M, N, dt, dev, 1.5) if act != "none" else None
    A, B, DY = a.double(), _kn(b, rows), dy.double()
    Z = z.double() if z is not None else torch.zeros_like(DY)
    own = act != "none" or dy32
    dz = Out(M, N, dt, dev) if own and not inplace else None
    dzt = None if not own else dz.t if dz else {"z": z, "dy": dy}[inplace]
    da, dbias = Out(M, K, f32 if da32 else dt, dev), torch.full((N + 8,), -77.0, device=dev)
    db = Out(*((N, K) if rows else (K, N)), f32 if db32 else dt, dev)
    kernels.linear_backward(dy, a, b, z=z, dz=dzt, da=da.t, db=db.t, dbias=dbias[:N], act=act, b_trans=rows)
    torch.cuda.synchronize()
    DZ = DY * act_grad64(Z, act)
    e32 = DY.abs() * grad_error(Z, act) + DZ.abs() * 2.0 ** -23  # dz before its rounding
    e16 = e32 + half_ulp(DZ, dt) if own else torch.zeros_like(DZ)
    if dz:
        dz.check("dz", DZ, e16)
    _check_product("da", da, DZ, B.t(), e16, None, N, da.t.dtype)
    if rows:
        _check_product("db", db, DZ.t(), A, e16.t(), None, M, db.t.dtype)
    else:
        _check_product("db", db, A.t(), DZ, None, e16, M, db.t.dtype)
    # fp32 sums of M values: each add rounds by 2^-24 of a partial sum.
    want, tol = DZ.sum(0), e32.sum(0) + DZ.abs().sum(0) * (M / 8 + 40) * 2.0 ** -24
    assert bool(((dbias[:N].double() - want).abs() <= tol).all())
    assert bool((dbias[N:] == -77.0).all())
    assert kernels.wait_status(clear=True) == 0


@pytest.mark.parametrize("dtype,rows,act,dx32,dw32,inplace", [
    ("bf16", True, "silu", False, False, False), ("fp16", False, "gelu_tanh", True, False, True),
    ("bf16", False, "gelu", False, True, False), ("fp16", True, "relu", True, True, True)])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gated_backward(dev, cudair, M, N, K, dtype, rows, act, dx32, dw32, inplace):
    import torch
    from cudair import kernels
    dt, f32 = _dt(dtype), torch.float32
    g = _gen(dev, M, N, K, 3)
    x, wg, wu = normal(g, M, K, dt, dev), _weight(g, N, K, dt, dev, rows), _weight(g, N, K, dt, dev, rows)
    gg, uu, dh = normal(g, M, N, dt, dev, 1.5), normal(g, M, N, dt, dev), normal(g, M, N, dt, dev)
    X, WG, WU, G, U, DH = x.double(), _kn(wg, rows), _kn(wu, rows), gg.double(), uu.double(), dh.double()
    dg, du = (None, None) if inplace else (Out(M, N, dt, dev), Out(M, N, dt, dev))
    dx = Out(M, K, f32 if dx32 else dt, dev)
    dwg, dwu = (Out(*((N, K) if rows else (K, N)), f32 if dw32 else dt, dev) for _ in range(2))
    # In place: dg over u and du over g, the crossing the documentation allows.
    kernels.gated_backward(dh, x, wg, wu, gg, uu, uu if inplace else dg.t, gg if inplace else du.t, dx=dx.t,
                           dwg=dwg.t, dwu=dwu.t, act=act, b_trans=rows)
    torch.cuda.synchronize()
    DG, DU = DH * U * act_grad64(G, act), DH * act64(G, act)
    eg = (DH * U).abs() * grad_error(G, act) + DG.abs() * 2.0 ** -22 + half_ulp(DG, dt)
    eu = DH.abs() * act_error(G, 0 * G, act) + DU.abs() * 2.0 ** -23 + half_ulp(DU, dt)
    if not inplace:
        dg.check("dg", DG, eg)
        du.check("du", DU, eu)
    pg, pu = DG.abs() @ WG.abs().t(), DU.abs() @ WU.abs().t()
    want = DG @ WG.t() + DU @ WU.t()
    dx.check("dx", want, half_ulp(want, dx.t.dtype) + eg @ WG.abs().t() + eu @ WU.abs().t() +
             sum_error(pg + pu, 2 * N + 128))
    for name, out, D, e in (("dwg", dwg, DG, eg), ("dwu", dwu, DU, eu)):
        if rows:
            _check_product(name, out, D.t(), X, e.t(), None, M, out.t.dtype)
        else:
            _check_product(name, out, X.t(), D, None, e, M, out.t.dtype)
    assert kernels.wait_status(clear=True) == 0


def test_empty_sizes(dev, cudair):
    import torch
    from cudair import kernels
    bf = torch.bfloat16
    t = lambda *s: torch.randn(*s, device=dev).to(bf)  # noqa: E731
    # K = 0: D = act(bias) + residual, H = 0.
    bias, r = torch.randn(24, device=dev), t(5, 24)
    for M in (5, 300):
        r, d, z = t(M, 24), torch.empty(M, 24, dtype=bf, device=dev), torch.empty(M, 24, dtype=bf, device=dev)
        kernels.linear(t(M, 0), t(0, 24), d, bias=bias, residual=r, z=z, act="relu")
        assert torch.equal(d, (torch.relu(bias) + r.float()).to(bf)) and torch.equal(z, bias.to(bf).expand(M, 24))
        h = torch.ones(M, 24, dtype=bf, device=dev)
        kernels.gated(t(M, 0), t(24, 0), t(24, 0), h, b_trans=True)
        assert not bool(h.any())
    # M = 0: no rows to write, and the weights' gradients are empty sums.
    e = t(0, 24)
    kernels.linear(t(0, 16), t(16, 24), e)
    kernels.gated(t(0, 16), t(16, 24), t(16, 24), e)
    db, dbias = torch.ones(16, 24, device=dev), torch.ones(24, device=dev)
    kernels.linear_backward(e, t(0, 16), t(16, 24), db=db, dbias=dbias)
    assert not bool(db.any()) and not bool(dbias.any())
    dwg, dwu = torch.ones(16, 24, dtype=bf, device=dev), torch.ones(16, 24, dtype=bf, device=dev)
    kernels.gated_backward(e, t(0, 16), t(16, 24), t(16, 24), e, e, e, e, dx=t(0, 16), dwg=dwg, dwu=dwu)
    assert not bool(dwg.any()) and not bool(dwu.any())
    # N = 0: dA and dX are empty sums.
    da, dx = torch.ones(5, 16, device=dev), torch.ones(5, 16, dtype=bf, device=dev)
    n = t(5, 0)
    kernels.linear_backward(n, t(5, 16), t(16, 0), da=da)
    kernels.gated_backward(n, t(5, 16), t(16, 0), t(16, 0), n, n, n, n, dx=dx)
    assert not bool(da.any()) and not bool(dx.any())
    # K = 0 leaves dbias alone to compute.
    kernels.linear_backward(t(5, 24).fill_(0.5), t(5, 0), t(0, 24), dbias=dbias)
    assert bool((dbias == 2.5).all())
    assert kernels.wait_status(clear=True) == 0


@pytest.mark.parametrize("M", [3, 100, 300])
def test_nan_and_inf_stay_in_their_row_and_column(dev, cudair, M):
    import torch
    from cudair import kernels
    N, K = 200, 96
    a, b = torch.randn(M, K, device=dev).half(), torch.randn(K, N, device=dev).half()
    d, z = torch.empty(M, N, device=dev), torch.empty(M, N, dtype=torch.float16, device=dev)
    kernels.linear(a, b, d, z=z, act="gelu")
    a2, b2 = a.clone(), b.clone()
    a2[M // 2, 5], b2[7, 130] = float("nan"), float("inf")
    d2 = torch.empty_like(d)
    kernels.linear(a2, b2, d2, act="gelu")
    clean = torch.ones(M, N, dtype=torch.bool, device=dev)
    clean[M // 2], clean[:, 130] = False, False
    assert torch.equal(d2[clean], d[clean]) and bool(d2[M // 2].isnan().all())
    assert not bool(d2[:, 130].isfinite().logical_and(a2[:, 7] > 0).any())
    # A NaN passes relu, and activations far out reach their limits.
    big = torch.tensor([[-6e4, -300.0, -0.0, 0.0, 300.0, 6e4, float("nan"), float("inf")]], device=dev).half()
    one = torch.eye(8, device=dev).half()
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        out = torch.empty(8, 8, device=dev)
        x = torch.diag(torch.nan_to_num(big[0].float(), nan=1.0, posinf=1.0)).half()
        kernels.linear(x, one, out, act=act)
        got = out.diagonal()[:6]
        assert bool((got[:4] == 0).all()) and bool((got[4:] == big[0, 4:6].float()).all()), (act, got)
        y = torch.empty(1, 8, device=dev)
        kernels.linear(big[:, 6:7].expand(1, 8).contiguous(), one, y, act=act)
        assert bool(y.isnan().all())
        # ... and their slopes 0 and 1.
        dz, dy = torch.empty(1, 8, dtype=torch.float16, device=dev), torch.ones(1, 8, device=dev).half()
        zz = torch.tensor([[-6e4, -3e4, -300.0, -100.0, 100.0, 300.0, 3e4, 6e4]], device=dev).half()
        kernels.linear_backward(dy, one[:1], one, z=zz, dz=dz, da=torch.empty_like(dz), act=act)
        assert dz[0].tolist() == [0, 0, 0, 0, 1, 1, 1, 1], (act, dz)
    # An infinite pre-activation stays infinite.
    k0, inf = torch.zeros(M, 0, device=dev).half(), torch.full((8,), float("inf"), device=dev)
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        y = torch.empty(M, 8, device=dev)
        kernels.linear(k0, torch.zeros(0, 8, device=dev).half(), y, bias=inf, act=act)
        assert bool((y == float("inf")).all()), act
    zz = torch.full((1, 8), 3e38, device=dev).bfloat16()
    dz = torch.empty_like(zz)
    for sign in (1, -1):
        for act in ("silu", "gelu", "gelu_tanh"):
            kernels.linear_backward(torch.ones_like(zz), one[:1].bfloat16(), one.bfloat16(), z=sign * zz, dz=dz,
                                    da=torch.empty_like(zz), act=act)
            assert bool((dz == (1 if sign > 0 else 0)).all()), (act, sign, dz)


@pytest.mark.parametrize("M", [5, 77, 200])
def test_residual_in_place_and_fused_weights(dev, cudair, M):
    """D over the residual's memory, and Wg, Wu as halves of one array."""
    import torch
    from cudair import kernels
    g = _gen(dev, M, 4)
    K, F = 264, 520
    x = normal(g, M, K, torch.bfloat16, dev)
    for rows in (False, True):
        both = normal(g, 2 * F, K, torch.bfloat16, dev, K ** -0.5) if rows else \
            normal(g, K, 2 * F, torch.bfloat16, dev, K ** -0.5)
        wg, wu = (both[:F], both[F:]) if rows else (both[:, :F], both[:, F:])
        h, h2 = (torch.empty(M, F, dtype=torch.bfloat16, device=dev) for _ in range(2))
        kernels.gated(x, wg, wu, h, b_trans=rows)
        kernels.gated(x, wg.contiguous(), wu.contiguous(), h2, b_trans=rows)
        assert torch.equal(h, h2)
        wd = normal(g, K, F, torch.bfloat16, dev, F ** -0.5) if rows else normal(g, F, K, torch.bfloat16, dev)
        stream = torch.randn(M, K, device=dev)
        d = torch.empty_like(stream)
        kernels.linear(h, wd, d, residual=stream, b_trans=rows)
        kernels.linear(h, wd, stream, residual=stream, b_trans=rows)
        assert torch.equal(d, stream)


@pytest.mark.parametrize("M,K,F,rows", [(3, 256, 520, True), (70, 264, 640, False), (300, 512, 1032, True)])
def test_feed_forward_layer(dev, cudair, M, K, F, rows):
    """The four operators as the layer y = x + (silu(x Wg) * (x Wu)) Wd + bd and
    its backward pass: against the chain rule in 64 bits, and the gradients'
    directional derivatives against central differences of the 64-bit layer."""
    import torch
    from cudair import kernels
    bf = torch.bfloat16
    gen = _gen(dev, M, K, F)
    x = normal(gen, M, K, bf, dev)
    wg, wu = (_weight(gen, F, K, bf, dev, rows) for _ in range(2))
    wd = _weight(gen, K, F, bf, dev, rows)
    bd, dy = torch.randn(K, generator=gen, device=dev), normal(gen, M, K, bf, dev)
    new = lambda r, c: torch.empty(r, -(-c // 8) * 8, dtype=bf, device=dev)[:, :c]  # noqa: E731
    h, g, u, y = new(M, F), new(M, F), new(M, F), new(M, K)
    kernels.gated(x, wg, wu, h, g=g, u=u, b_trans=rows)
    kernels.linear(h, wd, y, bias=bd, residual=x, b_trans=rows)
    dh, dg, du, dx = new(M, F), new(M, F), new(M, F), new(M, K)
    dwg, dwu, dwd = (new(*w.shape) for w in (wg, wu, wd))
    dbd = torch.empty(K, device=dev)
    kernels.linear_backward(dy, h, wd, da=dh, db=dwd, dbias=dbd, b_trans=rows)
    kernels.gated_backward(dh, x, wg, wu, g, u, dg, du, dx=dx, dwg=dwg, dwu=dwu, b_trans=rows)
    torch.cuda.synchronize()
    assert kernels.wait_status(clear=True) == 0

    def layer(x, wg, wu, wd, bd):
        mm = (lambda p, w: p @ w.t()) if rows else (lambda p, w: p @ w)
        gate = mm(x, wg)
        return x + mm(gate / (1 + torch.exp(-gate)) * mm(x, wu), wd) + bd

    leaves = [t.double().clone().requires_grad_() for t in (x, wg, wu, wd, bd)]
    want_y = layer(*leaves)
    want = torch.autograd.grad((want_y * dy.double()).sum(), leaves)
    # The residual's gradient is dy itself; the rest of dx is the gated pair's.
    got = [dx.double() + dy.double(), dwg.double(), dwu.double(), dwd.double(), dbd.double()]
    # Up to four roundings to 8 bits (h or g, u; dh; dg, du; the result), each
    # within 2^-9 of a value and independent: 4 x 2^-9 of the norm.
    want_y = want_y.detach()
    assert float((y.double() - want_y).norm() / want_y.norm()) <= 2 * 2.0 ** -9
    for name, p, q in zip(("dx", "dwg", "dwu", "dwd", "dbd"), got, want):
        rel = float((p - q).norm() / q.norm())
        assert rel <= 4 * 2.0 ** -9, (name, rel)
    # Differences: along a random direction scaled like the leaf, h = 1e-4, so
    # the central difference's own error (h^2) is far below the roundings'.
    with torch.no_grad():
        for i, p in enumerate(got):
            leaf = leaves[i]
            # Along the gradient itself, so that the derivative does not cancel.
            v = want[i] / want[i].norm() * leaf.norm()
            step = 1e-4
            ends = [layer(*[t + s * step * v if j == i else t for j, t in enumerate(leaves)]) for s in (1, -1)]
            slope = float(((ends[0] - ends[1]) * dy.double()).sum()) / (2 * step)
            mine = float((p * v).sum())
            assert abs(mine - slope) <= 4 * 2.0 ** -9 * abs(slope), (i, mine, slope)


@pytest.mark.parametrize("M", [4, 90, 300])
def test_streams_graphs_and_repeats(dev, cudair, M):
    """Calls on two streams at once, captured into two graphs and replayed
    together, with and without programmatic launches: bit for bit the same as
    one after the other."""
    import torch
    from cudair import kernels
    bf = torch.bfloat16
    gen = _gen(dev, M, 9)
    K, F = 512, 1536

    def problem():
        return dict(x=normal(gen, M, K, bf, dev), wg=_weight(gen, F, K, bf, dev, True),
                    wu=_weight(gen, F, K, bf, dev, True), wd=_weight(gen, K, F, bf, dev, True),
                    h=torch.empty(M, F, dtype=bf, device=dev), g=torch.empty(M, F, dtype=bf, device=dev),
                    u=torch.empty(M, F, dtype=bf, device=dev), y=torch.empty(M, K, dtype=bf, device=dev),
                    dh=torch.empty(M, F, dtype=bf, device=dev), dx=torch.empty(M, K, dtype=bf, device=dev),
                    dwg=torch.empty(F, K, dtype=bf, device=dev), dwu=torch.empty(F, K, dtype=bf, device=dev),
                    dwd=torch.empty(K, F, dtype=bf, device=dev), db=torch.empty(K, device=dev))

    outs = ("h", "y", "dh", "dx", "dwg", "dwu", "dwd", "db")

    def run(p, stream=None):
        kernels.gated(p["x"], p["wg"], p["wu"], p["h"], g=p["g"], u=p["u"], b_trans=True, stream=stream)
        kernels.linear(p["h"], p["wd"], p["y"], residual=p["x"], b_trans=True, stream=stream)
        kernels.linear_backward(p["y"], p["h"], p["wd"], da=p["dh"], db=p["dwd"], dbias=p["db"], b_trans=True,
                                stream=stream)
        kernels.gated_backward(p["dh"], p["x"], p["wg"], p["wu"], p["g"], p["u"], p["g"], p["u"], dx=p["dx"],
                               dwg=p["dwg"], dwu=p["dwu"], b_trans=True, stream=stream)

    ps = [problem(), problem()]
    want = []
    for p in ps:
        run(p)
        torch.cuda.synchronize()
        want.append({k: p[k].clone() for k in outs})

    def check(what):
        torch.cuda.synchronize()
        for p, w in zip(ps, want):
            for k in outs:
                assert torch.equal(p[k], w[k]), (what, k)
                p[k].fill_(3.0)
        torch.cuda.synchronize()

    for p in ps:
        for k in outs:
            p[k].fill_(3.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for mode in (0, 1, 2):
        kernels.set_gemm_pdl(mode)
        try:
            for _ in range(3):
                for p, s in zip(ps, streams):
                    run(p, stream=s)
            check(f"streams, launch mode {mode}")
            graphs = []
            for p in ps:
                gr = torch.cuda.CUDAGraph()
                with torch.cuda.graph(gr):
                    run(p)
                graphs.append(gr)
            for gr, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    gr.replay()
                    gr.replay()
            check(f"graphs, launch mode {mode}")
        finally:
            kernels.set_gemm_pdl(0)
    assert kernels.wait_status(clear=True) == 0


def test_64_bit_offsets(dev, cudair):
    """Rows past 2^31 elements into a matrix, read and written."""
    import torch
    from cudair import kernels
    M, N, K = 9, 64, 64
    ld = 1 << 28  # row 8 starts at 2^31 elements
    bf = torch.bfloat16
    big = torch.empty(8 * ld + 256, dtype=bf, device=dev)
    x, y = big.as_strided((M, K), (ld, 1), 0), big.as_strided((M, N), (ld, 1), 64)
    x.copy_(torch.randn(M, K, device=dev))
    w = torch.randn(N, K, device=dev).to(bf)
    small = torch.empty(M, N, dtype=bf, device=dev)
    kernels.linear(x.contiguous(), w, small, act="silu", b_trans=True)
    kernels.linear(x, w, y, act="silu", b_trans=True)
    assert torch.equal(y, small)
    dz = big.as_strided((M, N), (ld, 1), 128)
    db, db2, dz2 = (torch.empty(N, K, device=dev), torch.empty(N, K, device=dev),
                    torch.empty(M, N, dtype=bf, device=dev))
    kernels.linear_backward(y, x, w, z=y, dz=dz, db=db, act="silu", b_trans=True)
    kernels.linear_backward(small, x.contiguous(), w, z=small, dz=dz2, db=db2, act="silu", b_trans=True)
    assert torch.equal(dz, dz2) and torch.equal(db, db2)


def test_many_sizes_at_once(dev, cudair):
    """Calls of every tile height, plain and gated, kept in flight together on
    four streams: each as when it runs alone."""
    import torch
    from cudair import kernels
    bf = torch.bfloat16
    gen = _gen(dev, 77)
    calls = []
    for M in (1, 20, 40, 64, 90, 128, 200, 500):
        for K, N, gated in ((2048, 640, False), (512, 1408, True), (1088, 4096, False)):
            x, w, w2 = normal(gen, M, K, bf, dev), _weight(gen, N, K, bf, dev, True), _weight(gen, N, K, bf, dev, True)
            y = torch.empty(M, N, dtype=bf, device=dev)

            def call(stream, x=x, w=w, w2=w2, y=y, gated=gated):
                if gated:
                    kernels.gated(x, w, w2, y, b_trans=True, stream=stream)
                else:
                    kernels.linear(x, w, y, act="gelu", b_trans=True, stream=stream)
            calls.append((call, y))
    want = []
    for call, y in calls:
        call(None)
        torch.cuda.synchronize()
        want.append(y.clone())
        y.fill_(9.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for turn in range(6):
        for i, (call, _) in enumerate(calls):
            call(streams[(i + turn) % 4] if turn % 2 else streams[i % 4])
        torch.cuda.synchronize()
        for (_, y), w in zip(calls, want):
            assert torch.equal(y, w)
            y.fill_(9.0)
        torch.cuda.synchronize()
    assert kernels.wait_status(clear=True) == 0


_CAPTURE = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from cudair import kernels
bf, dev = torch.bfloat16, "cuda"
r = lambda *s: torch.randn(*s, device=dev).to(bf)
M, N, K = (40, 256, 128) if sys.argv[2] == "few" else (1304, 1104, 1200)
x, w, w2, y, z, g, u, h = r(M, K), r(N, K), r(N, K), r(M, N), r(M, N), r(M, N), r(M, N), r(M, N)
outs = [torch.empty_like(t) for t in (x, w, w2, x, w, y, y, y)]
db = torch.empty(N, device=dev)
def run():
    kernels.gated(x, w, w2, outs[5], act="silu", b_trans=True)
    kernels.linear(x, w, outs[6], act="gelu", b_trans=True)
    kernels.linear_backward(y, x, w, z=z, dz=outs[7], da=outs[0], db=outs[1], dbias=db, act="gelu", b_trans=True)
    kernels.gated_backward(h, x, w, w2, g, u, g, u, dx=outs[3], dwg=outs[2], dwu=outs[4], b_trans=True)
torch.cuda.synchronize()
g0, u0 = g.clone(), u.clone()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    run()  # the library's first call in this process
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in outs + [db]]
g.copy_(g0); u.copy_(u0)
run()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, outs + [db]))
assert kernels.wait_status() == 0
print("captured")
"""


@pytest.mark.parametrize("size", ["few", "many"])
def test_first_call_may_be_captured(dev, cudair, size):
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _CAPTURE, os.path.join(here, "cuda-ir.go_b200"), size],
                       capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_wrapper_refusals(dev, cudair):
    import torch
    from cudair import kernels
    from cudair._lib import CudairError
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device=dev)  # noqa: E731
    a, b, d = h(4, 16), h(16, 24), h(4, 24)
    for message, call in [
            ("a must be a float16 or bfloat16 tensor", lambda: kernels.linear(a.float(), b, d)),
            ("a must be a float16 or bfloat16 tensor", lambda: kernels.linear(None, b, d)),
            ("a and b must be matrices", lambda: kernels.linear(a, None, d)),
            ("b must be torch.float16, got torch.bfloat16", lambda: kernels.linear(a, b.bfloat16(), d)),
            ("b must be 16 x 20", lambda: kernels.linear(a, h(18, 20), d)),
            ("d must be 4 x 24", lambda: kernels.linear(a, b, h(4, 25))),
            ("d must be torch.float16 or torch.float32", lambda: kernels.linear(a, b, d.bfloat16())),
            ("d needs unit inner stride", lambda: kernels.linear(a, b, h(24, 4).t())),
            ("d must be a CUDA tensor", lambda: kernels.linear(a, b, d.cpu())),
            ("pitch 25 of d must be a multiple of 8", lambda: kernels.linear(a, b, h(4, 25)[:, :24])),
            ("bias must have 24 consecutive values", lambda: kernels.linear(a, b, d, bias=h(23))),
            ("bias must have 24 consecutive values", lambda: kernels.linear(a, b, d, bias=h(48)[::2])),
            ("residual must be torch.float16", lambda: kernels.linear(a, b, d, residual=d.float())),
            ("act must be one of none, relu, gelu, gelu_tanh, silu", lambda: kernels.linear(a, b, d, act="tanh")),
            ("d lies over another matrix", lambda: kernels.linear(h(4, 24), h(24, 24), d, z=d)),
            ("g and u are given together", lambda: kernels.gated(a, b, b, d, g=h(4, 24))),
            ("wu must be 16 x 24", lambda: kernels.gated(a, b, h(16, 25), d)),
            (r"nil pointer \(dz\)", lambda: kernels.linear_backward(d, a, b, z=h(4, 24), da=h(4, 16), act="relu")),
            ("dz must be nil", lambda: kernels.linear_backward(d, a, b, dz=h(4, 24), da=h(4, 16))),
            ("dbias must be torch.float32", lambda: kernels.linear_backward(d, a, b, dbias=h(24))),
            ("dwg and dwu are given together", lambda: kernels.gated_backward(
                d, a, b, b, h(4, 24), h(4, 24), h(4, 24), h(4, 24), dwg=h(16, 24)))]:
        with pytest.raises(CudairError, match=message):
            call()
    # One row needs no pitch of its own.
    kernels.linear(h(1, 15), h(15, 24), h(1, 24))
    torch.cuda.synchronize()

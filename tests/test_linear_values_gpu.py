"""The activations of the feed-forward operators value by value, against their
formulas in 64 bits, with bounds relative to the value: where an activation
is small (negative arguments) it is an output like any other.

How far an fp32 evaluation may be off, relative to the value (2^-24 is a
rounding; the hardware's 2^x is within 2^-22, its reciprocal within 2^-23):
  e^x    with x from n roundings is off by n 2^-24 |x| in its exponent;
  silu   z / (1 + e^-z): x = -z from two roundings (the constant log2 e, the
         product), then 2^x, a sum, a reciprocal and a product: 2 |z| 2^-24 + 2^-21;
  gelu_tanh  x = 2y = 2 sqrt(2/pi) (z + 0.044715 z^3) with constants of up to
         five roundings and three more: 8 |x| 2^-24 + 2^-21;
  gelu   |z| E R, E = e^(-z^2 / 2) from three roundings of z^2 / 2; R a fitted
         polynomial, within 2^-20 of the function when evaluated in fp32 with an exact
         reciprocal, 2^-22 more with the hardware's (R's slope in it is below two);
         the rest 2^-21: 1.5 z^2 2^-24 + 2^-20 + 2^-21 + 2^-22.
Each output adds half a step of its type, or half its smallest subnormal; an
exponential or its reciprocal below 2^-126 becomes 0, which is |z| 2^-126 <= 2^-122
of the value."""
import math

import pytest

pytestmark = pytest.mark.gpu

ACTS = ("silu", "gelu", "gelu_tanh")
TINY = {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -134, "float32": 2.0 ** -150}


def formula(z, act):
    import torch
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def relative(z, act):
    u = z.abs()
    if act == "silu":
        return 2 * u * 2.0 ** -24 + 2.0 ** -21
    if act == "gelu":
        return 1.5 * z * z * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -21 + 2.0 ** -22
    return 8 * 2 * math.sqrt(2 / math.pi) * (u + 0.044715 * u ** 3) * 2.0 ** -24 + 2.0 ** -21


def off(got, z, act, extra=0.0):
    """got against act(z), as a fraction of what is allowed; its largest value and where."""
    import torch
    want = formula(z, act)
    tol = want.abs() * (relative(z, act) + extra + torch.finfo(got.dtype).eps / 2) + \
        TINY[str(got.dtype).split(".")[1]] + 2.0 ** -122
    ratio = (got.double() - want).abs() / tol
    i = int(ratio.argmax())
    return float(ratio[i]), float(z[i]), float(got[i]), float(want[i])


@pytest.mark.parametrize("M", [3, 300])
@pytest.mark.parametrize("out", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("act", ACTS)
def test_forward_values_keep_their_relative_accuracy(dev, cudair, act, out, M):
    """z = the bias, 65536 values over [-12, 0] and over [0, 12]."""
    import torch
    from cudair import kernels
    dt = getattr(torch, out)
    t16 = torch.float16 if dt is torch.float16 else torch.bfloat16
    N = 65536
    for z in (torch.linspace(-12, 0, N, device=dev), torch.linspace(0, 12, N, device=dev)):
        d = torch.empty(M, N, dtype=dt, device=dev)
        kernels.linear(torch.empty(M, 0, dtype=t16, device=dev), torch.empty(0, N, dtype=t16, device=dev), d, bias=z,
                       act=act)
        assert torch.equal(d, d[:1].expand(M, N))
        ratio = off(d[0], z.double(), act)
        assert ratio[0] <= 1, ratio
    assert kernels.wait_status(clear=True) == 0


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("act", ACTS)
def test_backward_values_keep_their_relative_accuracy(dev, cudair, act, dtype):
    """The gated gradient's dU = dH act(G) with dH = 1, at every G of the type in [-12, 12]."""
    import torch
    from cudair import kernels
    dt = getattr(torch, dtype)
    every = torch.arange(-32768, 32768, device=dev, dtype=torch.int32).to(torch.int16).view(dt)
    g = every[every.abs() <= 12]
    n = g.numel() // 8 * 8
    g = g[:n].reshape(1, n).contiguous()
    one, x = torch.ones_like(g), torch.empty(1, 0, dtype=dt, device=dev)
    w = torch.empty(0, n, dtype=dt, device=dev)
    dg, du = torch.empty_like(g), torch.empty_like(g)
    kernels.gated_backward(one, x, w, w, g, one, dg, du, act=act)
    ratio = off(du[0], g[0].double(), act)
    assert ratio[0] <= 1, ratio


@pytest.mark.parametrize("M", [3, 300])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("act", ACTS + ("relu", "none"))
def test_infinite_and_far_arguments_reach_the_limits(dev, cudair, act, dtype, M):
    """Values: 0 and z; derivatives: 0 and 1; a NaN stays one.  The same for the largest finite
    arguments, in the forward's epilogue (z by the bias) and in the gradient's element-wise step."""
    import torch
    from cudair import kernels
    dt, inf, nan = getattr(torch, dtype), float("inf"), float("nan")
    far = float(torch.finfo(dt).max)
    z = torch.tensor([-inf, -far, -far / 4, far / 4, far, inf, nan, -100], device=dev)
    low = [0.0] * 3 if act != "none" else [-inf, -far, -far / 4]
    want = torch.tensor(low + [far / 4, far, inf, nan, 0 if act != "none" else -100], device=dev)
    slope = torch.tensor([0.0 if act != "none" else 1.0] * 3 + [1.0] * 3, device=dev)
    same = lambda p, q: bool(((p == q) | (p.isnan() & q.isnan())).all())  # noqa: E731
    d, zz = torch.empty(M, 8, device=dev), torch.empty(M, 8, dtype=dt, device=dev)
    kernels.linear(torch.empty(M, 0, dtype=dt, device=dev), torch.empty(0, 8, dtype=dt, device=dev), d, bias=z,
                   z=zz, act=act)
    assert same(d, want.expand(M, 8)), d[0]
    assert same(zz, z.to(dt).expand(M, 8)), zz[0]
    # linear_backward: dZ = act'(Z); gated_backward: dG = act'(G), dU = act(G), with dH = U = 1.
    ones = torch.ones_like(zz)
    x, w = torch.empty(M, 0, dtype=dt, device=dev), torch.empty(0, 8, dtype=dt, device=dev)
    dg, du, dz = (torch.empty_like(zz) for _ in range(3))
    kernels.gated_backward(ones, x, w, w, zz, ones, dg, du, act=act)
    assert same(du.float(), want.to(dt).float().expand(M, 8)), du[0]
    grads = [dg]
    if act != "none":
        kernels.linear_backward(ones, x, w, z=zz, dz=dz, act=act)
        grads.append(dz)
    for g in grads:
        assert torch.equal(g[:, :6].float(), slope.expand(M, 6)), g[0]
        assert act == "none" or act == "relu" or bool(g[:, 6].isnan().all())
    assert kernels.wait_status(clear=True) == 0

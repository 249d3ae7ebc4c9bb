"""The feed-forward operators' definitions in 64 bits, and how far 16-bit or
fp32 results may be from them.

Error model, used by every bound below:
  * a product of two 16-bit values is exact in fp32; a sum of K of them is
    built by K / 16 matrix instructions, each of which may lose two units in
    the last place (2^-23 relative each) of the magnitude it works at, which
    is at most S = sum |a||b|:  |sum error| <= (K / 16 + 4) 2^-22 S;
  * the split sums joined afterwards lose less than the four extra steps above;
  * an activation's slope is at most 1.13 in magnitude, and its fp32
    evaluation is within 2^-20 of its value (exp, division and normcdf are
    within a few 2^-24 of theirs, with an argument error of |z| 2^-22 in the
    exponent for |z| up to 16), plus 2^-22 |z| where two terms cancel;
  * each rounding to a type is off by at most eps / 2 of the value, or half
    its smallest subnormal.
"""
import math

import torch

SLOPE = 1.13
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def act64(z, act):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2))
    return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def act_grad64(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    with torch.enable_grad():
        x = z.detach().clone().requires_grad_()
        return torch.autograd.grad(act64(x, act).sum(), x)[0]


def half_ulp(ref, dtype):
    return ref.abs() * (torch.finfo(dtype).eps / 2) + TINY[dtype]


def sum_error(absprod, K):
    return absprod * ((K / 16 + 4) * 2.0 ** -22)


def act_error(z, dz, act):
    """Of act(z) for a z that is off by dz."""
    if act == "none":
        return dz
    return SLOPE * dz + (act64(z, act).abs() + z.abs() / 4) * 2.0 ** -20


def grad_error(z, act):
    """Of act'(z) at an exact z: values up to 1.13, terms up to |z| that cancel."""
    if act in ("none", "relu"):
        return torch.zeros_like(z)
    return (1 + z.abs().clamp(max=16)) * 2.0 ** -19


def padded(rows, cols, dtype, dev, pad=8, lead=0, fill=float("nan")):
    """A rows x cols view of a larger array: pitch rounded up to 8 elements plus
    `pad`, starting `lead` elements in, the rest holding `fill`."""
    ld = -(-cols // 8) * 8 + pad
    whole = torch.full((lead + max(rows, 1) * ld + 8,), fill, dtype=dtype, device=dev)
    return whole.as_strided((rows, cols), (ld, 1), lead), whole


def normal(g, rows, cols, dtype, dev, std=1.0, pad=8, lead=0):
    v, _ = padded(rows, cols, dtype, dev, pad, lead)
    v.copy_(torch.randn(rows, cols, generator=g, device=dev) * std)
    return v


class Out:
    """An output inside a larger array of sentinels that must stay as they are."""

    def __init__(self, rows, cols, dtype, dev, pad=8, lead=0):
        self.t, self.whole = padded(rows, cols, dtype, dev, pad, lead, fill=-77.0)
        self.t.fill_(float("nan"))

    def check(self, name, ref, tol):
        got = self.t.double()
        bad = ~((got - ref).abs() <= tol)
        if bool(bad.any()):
            i = int(bad.flatten().nonzero()[0])
            r, c = divmod(i, ref.shape[1])
            raise AssertionError(f"{name}: {int(bad.sum())} of {ref.numel()} values off; [{r}, {c}] is "
                                 f"{float(got[r, c])}, want {float(ref[r, c])} +- {float(tol[r, c])}")
        keep = self.t.clone()
        self.t.fill_(-77.0)
        assert bool((self.whole == -77.0).all()), f"{name}: values outside the matrix were written"
        self.t.copy_(keep)

"""What cudair_linear, cudair_gated and their gradients refuse, on CPU: the
arguments are checked before the driver is touched."""
import ctypes
import re

import pytest

from cudair import _lib

P = 0x7F0000000000  # a 16-byte aligned address; never dereferenced on CPU
BF16, B_T, D_F32, BIAS_16, DA_F32, DB_F32 = 0x1, 0x2, 0x10, 0x20, 0x40, 0x80


def _at(i):
    """The i-th of some separate arrays."""
    return P + (i << 20)


def _linear(**over):
    a = dict(a=_at(0), b=_at(1), bias=None, residual=None, d=_at(2), z=None, M=4, N=24, K=16, lda=16, ldb=24,
             ldres=0, ldd=24, ldz=0, act=0, flags=0)
    return "cudair_linear", _lib.LinearArgs(**{**a, **over})


def _gated(**over):
    a = dict(x=_at(0), wg=_at(1), wu=_at(2), h=_at(3), g=None, u=None, M=4, N=24, K=16, ldx=16, ldwg=24, ldwu=24,
             ldh=24, ldg=0, ldu=0, act=4, flags=0)
    return "cudair_gated", _lib.GatedArgs(**{**a, **over})


def _linear_backward(**over):
    a = dict(dy=_at(0), a=_at(1), b=_at(2), z=_at(3), dz=_at(4), da=_at(5), db=_at(6), dbias=_at(7), M=4, N=24,
             K=16, lddy=24, lda=16, ldb=24, ldz=24, lddz=24, ldda=16, lddb=24, act=2, flags=0)
    return "cudair_linear_backward", _lib.LinearBackwardArgs(**{**a, **over})


def _gated_backward(**over):
    a = dict(dh=_at(0), x=_at(1), wg=_at(2), wu=_at(3), g=_at(4), u=_at(5), dg=_at(6), du=_at(7), dx=_at(8),
             dwg=_at(9), dwu=_at(10), M=4, N=24, K=16, lddh=24, ldx=16, ldwg=24, ldwu=24, ldg=24, ldu=24, lddg=24,
             lddu=24, lddx=16, lddwg=24, lddwu=24, act=4, flags=0)
    return "cudair_gated_backward", _lib.GatedBackwardArgs(**{**a, **over})


@pytest.mark.parametrize("call,message", [
    (_linear(M=-1), "negative size"),
    (_linear(N=2 ** 31 - 1), "sizes must be at most"),
    (_linear(flags=0x8), "unknown flags 0x8"),
    (_linear(flags=DA_F32), "unknown flags 0x40"),
    (_linear(act=5), "unknown activation 5"),
    (_linear(a=None), r"nil pointer \(a\)"),
    (_linear(d=None), r"nil pointer \(d\)"),
    (_linear(b=P + 8), "b must be 16-byte aligned"),
    (_linear(d=P + 2), "d must be 16-byte aligned"),
    (_linear(lda=8), "pitch 8 of a is below its 16 columns"),
    (_linear(ldb=20), "pitch 20 of b is below its 24 columns"),
    (_linear(ldb=28), "pitch 28 of b must be a multiple of 8"),
    (_linear(flags=B_T, ldb=12), "pitch 12 of b is below its 16 columns"),
    (_linear(ldd=25), "pitch 25 of d must be a multiple of 8"),
    (_linear(flags=D_F32, ldd=26), "pitch 26 of d must be a multiple of 4"),
    (_linear(residual=P, ldres=8), "pitch 8 of residual is below"),
    (_linear(residual=_at(2), ldres=32), "a residual in D's memory needs D's pitch"),
    (_linear(z=P + 1, ldz=24), "z must be 16-byte aligned"),
    (_linear(bias=P + 2), "bias must be aligned"),
    (_linear(bias=P + 1, flags=BIAS_16), "bias must be aligned"),
    (_linear(ldd=1 << 40), "pitch 1099511627776 of d is too large"),
    (_gated(flags=D_F32), "unknown flags 0x10"),
    (_gated(wu=None), r"nil pointer \(wu\)"),
    (_gated(h=None), r"nil pointer \(h\)"),
    (_gated(g=P, ldg=24), "g and u are given together"),
    (_gated(u=P, ldu=24), "g and u are given together"),
    (_gated(g=P, u=P, ldg=24, ldu=23), "pitch 23 of u is below"),
    (_gated(ldwg=16), "pitch 16 of wg is below"),
    (_linear_backward(z=None), r"nil pointer \(z\)"),
    (_linear_backward(dz=None), r"nil pointer \(dz\)"),
    (_linear_backward(act=0), "dz must be nil"),
    (_linear_backward(act=0, flags=D_F32, dz=None), r"nil pointer \(dz\)"),
    (_linear_backward(dz=_at(0), lddz=32), "dz in dY's memory"),
    (_linear_backward(dz=_at(0), flags=D_F32), "dz in dY's memory"),
    (_linear_backward(dz=_at(3), lddz=32), "dz in z's memory"),
    (_linear_backward(b=None), r"nil pointer \(b\)"),
    (_linear_backward(a=None), r"nil pointer \(a\)"),
    (_linear_backward(ldda=8), "pitch 8 of da is below"),
    (_linear_backward(dbias=P + 2), "dbias must be 4-byte aligned"),
    (_gated_backward(dg=_at(7)), "dg and du share memory"),
    (_gated_backward(dg=None), r"nil pointer \(dg\)"),
    (_gated_backward(dwg=None), "dwg and dwu are given together"),
    (_gated_backward(dg=_at(0), lddg=32), "in an input's memory needs its pitch"),
    (_gated_backward(lddx=8), "pitch 8 of dx is below"),
    (_gated_backward(wg=None), r"nil pointer \(wg\)"),
    (_gated_backward(flags=BIAS_16), "unknown flags 0x20"),
    # An output over an input or another output, but for the allowed places.
    (_linear(d=_at(0)), "d lies over another"),
    (_linear(z=_at(2), ldz=24), "d lies over another"),
    (_linear(residual=P, ldres=24, z=P, ldz=24), "z lies over another"),
    (_gated(g=_at(3), u=_at(4), ldg=24, ldu=24), "h lies over another"),
    (_gated(g=_at(4), u=_at(4), ldg=24, ldu=24), "g lies over another"),
    (_gated(g=_at(5), u=_at(1), ldg=24, ldu=24), "u lies over another"),
    (_linear_backward(da=_at(1)), "da lies over another"),
    (_linear_backward(da=_at(4)), "dz lies over another"),
    (_linear_backward(db=_at(2)), "db lies over another"),
    (_linear_backward(dbias=_at(2)), "dbias lies over another"),
    (_linear_backward(dbias=_at(4), K=0), "dbias lies over another"),
    (_linear_backward(dbias=_at(6), M=0), "dbias lies over another"),
    (_gated_backward(dx=_at(1)), "dx lies over another"),
    (_gated_backward(dwu=_at(9)), "dwg lies over another"),
    (_gated_backward(dwu=_at(9), M=0), "dwg lies over another"),
    (_gated_backward(dwg=_at(2)), "dwg lies over another"),
    (_gated_backward(du=_at(8)), "du lies over another"),
    # Contractions that a bounded wait would not outlast.
    (_linear(K=2 ** 26 + 8, lda=2 ** 26 + 8), "contraction over 67108872 is too long"),
    (_gated(K=2 ** 27, ldx=2 ** 27), "contraction over 134217728 is too long"),
    (_linear_backward(M=2 ** 26 + 1), "contraction over 67108865 is too long"),
    (_gated_backward(M=2 ** 26 + 1), "contraction over 67108865 is too long"),
], ids=lambda v: v[0] if isinstance(v, tuple) else None)
def test_refusals(cudair, call, message):
    name, args = call
    rc = getattr(cudair.lib(), name)(ctypes.byref(args), None)
    op = name[len("cudair_"):]
    assert rc == _lib.ERR_INVALID
    assert re.search(f"^cudair: {op}: .*{message}", cudair.last_error()), cudair.last_error()


def test_nil_arguments_and_no_ops(cudair):
    L = cudair.lib()
    for name in ("cudair_linear", "cudair_linear_backward", "cudair_gated", "cudair_gated_backward"):
        assert getattr(L, name)(None, None) == _lib.ERR_INVALID and "nil arguments" in cudair.last_error()
    # Sizes of zero need no operands, and no device where nothing is written.
    for name, args in (_linear(M=0, a=None, d=None), _linear(N=0, b=None, d=None), _gated(M=0, x=None, h=None)):
        assert getattr(L, name)(ctypes.byref(args), None) == 0


def test_structs_match_the_header():
    """Field names, order and types of the ctypes structs."""
    text = re.sub(r"/\*.*?\*/", "", open(_lib.HEADER_PATH).read(), flags=re.S)
    for cls in (_lib.LinearArgs, _lib.LinearBackwardArgs, _lib.GatedArgs, _lib.GatedBackwardArgs):
        body = re.search(r"typedef struct %s \{(.*?)\}" % cls.__name__, text, re.S).group(1)
        want = []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            names = [n.strip() for n in decl.split(",")]
            kind, first = names[0].rsplit(None, 1) if "*" not in names[0] else ("ptr", names[0].split("*")[1])
            for n in [first] + names[1:]:
                want.append((n.strip("* "), "ptr" if "*" in decl else kind.strip()))
        kinds = {ctypes.c_void_p: "ptr", ctypes.c_int64: "int64_t", ctypes.c_uint32: "uint32_t"}
        assert [(n, kinds[t]) for n, t in cls._fields_] == want

"""Gradients of calls that need only some of their operands (a frozen weight, a
first layer without an input gradient): the operand that nothing needs may be
left out, and what is computed is what the whole call computes."""
import pytest

from linear_ref import normal
from test_linear_gpu import _gen, _weight

pytestmark = pytest.mark.gpu


def reordered(length):
    """How far two orders of one fp32 sum of `length` products may be apart: each within (length / 16 + 4) 2^-22 of
    the sum of magnitudes (linear_ref.py), which is below `length` for factors of unit variance."""
    return 2 * (length / 16 + 4) * 2.0 ** -22 * length


SIZES = [(5, 264, 136, True), (5, 264, 136, False), (300, 520, 264, True), (1300, 1032, 512, False)]


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("M,N,K,rows", SIZES)
def test_linear_backward(dev, cudair, M, N, K, rows, act):
    import torch
    from cudair import kernels
    bf = torch.bfloat16
    gen = _gen(dev, M, N, K, 41)
    a, b, dy = normal(gen, M, K, bf, dev), _weight(gen, N, K, bf, dev, rows), normal(gen, M, N, bf, dev)
    z = normal(gen, M, N, bf, dev) if act != "none" else None

    def call(a, b, want):
        o = {k: torch.full(s, 5.0, dtype=t, device=dev) for k, s, t in
             (("da", (M, K), bf), ("db", tuple(_weight(gen, N, K, bf, dev, rows).shape), torch.float32),
              ("dbias", (N,), torch.float32)) if k in want}
        dz = torch.empty(M, N, dtype=bf, device=dev) if act != "none" else None
        kernels.linear_backward(dy, a, b, z=z, dz=dz, act=act, b_trans=rows, **o)
        return o | ({"dz": dz} if dz is not None else {})

    whole = call(a, b, ("da", "db", "dbias"))
    for args, want in (((None, b), ("da", "dbias")), ((a, None), ("db", "dbias")), ((None, None), ("dbias",)),
                       ((None, b), ("da",)), ((a, None), ("db",)), ((None, None), ())):
        for k, t in call(*args, want).items():
            # Which products share a launch may differ, and with it the order of a sum; in bf16 that is a step.
            assert torch.allclose(t.double(), whole[k].double(), rtol=2.0 ** -7, atol=reordered(max(M, N))), (want, k)
            if k in ("dz", "dbias"):
                assert torch.equal(t, whole[k]), (want, k)
    for args, want, message in (((None, b), ("db",), "nil pointer .a."), ((a, None), ("da",), "nil pointer .b.")):
        with pytest.raises(cudair.CudairError, match=message):
            call(*args, want)
    assert kernels.wait_status(clear=True) == 0


@pytest.mark.parametrize("M,N,K,rows", SIZES)
def test_gated_backward(dev, cudair, M, N, K, rows):
    import torch
    from cudair import kernels
    dt = torch.float16
    gen = _gen(dev, M, N, K, 42)
    x, dh = normal(gen, M, K, dt, dev), normal(gen, M, N, dt, dev)
    wg, wu = (_weight(gen, N, K, dt, dev, rows) for _ in range(2))
    g, u = (normal(gen, M, N, dt, dev) for _ in range(2))

    def call(x, wg, wu, want):
        o = {k: torch.full(s, 5.0, device=dev) for k, s in
             (("dx", (M, K)), ("dwg", (N, K) if rows else (K, N)), ("dwu", (N, K) if rows else (K, N))) if k in want}
        dg, du = (torch.empty(M, N, dtype=dt, device=dev) for _ in range(2))
        kernels.gated_backward(dh, x, wg, wu, g, u, dg, du, b_trans=rows, **o)
        return o | {"dg": dg, "du": du}

    whole = call(x, wg, wu, ("dx", "dwg", "dwu"))
    for args, want in (((None, wg, wu), ("dx",)), ((x, None, None), ("dwg", "dwu")), ((None, None, None), ())):
        for k, t in call(*args, want).items():
            assert float((t.double() - whole[k].double()).abs().max()) <= reordered(max(M, 2 * N)), (want, k)
    for args, want, message in (((None, wg, wu), ("dwg", "dwu"), "nil pointer .x."),
                                ((x, None, wu), ("dx",), "nil pointer .wg."),
                                ((x, wg, None), ("dx",), "nil pointer .wu.")):
        with pytest.raises(cudair.CudairError, match=message):
            call(*args, want)
    assert kernels.wait_status(clear=True) == 0


def test_shapes_that_do_not_fit(dev, cudair):
    import torch
    from cudair import kernels
    h = lambda *s: torch.zeros(*s, dtype=torch.float16, device=dev)  # noqa: E731
    for message, call in [
            ("b must be 16 x 24", lambda: kernels.linear_backward(h(4, 24), h(4, 16), h(16, 32), da=h(4, 16))),
            ("a must be 4 x 16", lambda: kernels.linear_backward(h(4, 24), h(5, 16), None, db=h(16, 24))),
            ("db must be 16 x 24", lambda: kernels.linear_backward(h(4, 24), h(4, 16), None, db=h(24, 16))),
            ("dy must be a matrix", lambda: kernels.linear_backward(h(24), h(4, 16), None, db=h(16, 24))),
            ("dy must be a float16 or bfloat16", lambda: kernels.linear_backward(h(4, 24).float(), None, None)),
            ("dh must be a float16 or bfloat16", lambda: kernels.gated_backward(None, h(4, 16), *[h(4, 24)] * 6)),
            ("the weight must be a matrix", lambda: kernels.gated_backward(h(4, 24), h(4, 16), h(16), h(16), h(4, 24),
                                                                          h(4, 24), h(4, 24), h(4, 24), dx=h(4, 16))),
            ("wu must be 16 x 24", lambda: kernels.gated_backward(h(4, 24), None, h(16, 24), h(16, 16), h(4, 24),
                                                                 h(4, 24), h(4, 24), h(4, 24), dx=h(4, 16)))]:
        with pytest.raises(cudair.CudairError, match=message):
            call()

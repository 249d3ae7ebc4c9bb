"""Both kernels of the feed-forward operators, each pinned by
cudair_set_linear_kernel, and CTA pairs with every tile width, against 64 bits:
the checks and tolerances are those of test_linear_gpu.py, where the
sizes decide which kernel runs.

A pair's ring holds seven k-blocks of 64 (one accumulator block per tile) or four (two
blocks: widths from 384), so 200, 260, 520 and 1100 lie below, at, and past one and two
ring-fulls of both.  2049 x 4103 and 4100 x 2600 are more tiles than the 74 pairs of the device
at every width, so accumulators change hands under a running epilogue."""
import contextlib

import pytest

import test_linear_gpu as plain
from linear_ref import normal

pytestmark = pytest.mark.gpu

SPLIT, PAIRS = 1, 2
KERNELS = [(SPLIT, 0)] + [(PAIRS, w) for w in (192, 224, 256, 384, 448, 512)]
NAMES = ["split"] + [f"pairs-{w}" for _, w in KERNELS[1:]]
SHAPES = [(2049, 4103, 200), (4100, 2600, 1100), (4352, 2560, 64), (300, 70, 520), (1, 515, 260), (3000, 1031, 0)]
GRADIENT_SHAPES = [(4100, 2600, 1100), (130, 4100, 4000), (300, 515, 1029), (1, 8, 8)]


@contextlib.contextmanager
def pinned(kernel, width):
    from cudair import kernels
    kernels.set_linear_kernel(kernel, width)
    try:
        yield
    finally:
        kernels.set_linear_kernel(0)


@pytest.mark.parametrize("kernel", KERNELS, ids=NAMES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear(dev, cudair, M, N, K, kernel):
    for form in plain.FORMS:
        with pinned(*kernel):
            plain.test_linear(dev, cudair, M, N, K, form)


@pytest.mark.parametrize("kernel", [k for k in KERNELS if k[1] not in (224, 448)],
                         ids=[n for n in NAMES if n[-3:] not in ("224", "448")])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gated(dev, cudair, M, N, K, kernel):
    for form in [("bf16", True, "silu", True, 8, 0), ("fp16", False, "gelu_tanh", False, 0, 8),
                 ("bf16", False, "gelu", True, 24, 8), ("fp16", True, "relu", True, 0, 0)]:
        with pinned(*kernel):
            plain.test_gated(dev, cudair, M, N, K, *form)


@pytest.mark.parametrize("kernel", KERNELS, ids=NAMES)
@pytest.mark.parametrize("M,N,K", GRADIENT_SHAPES)
def test_linear_backward(dev, cudair, M, N, K, kernel):
    for form in [("bf16", True, "gelu_tanh", False, False, False, None), ("fp16", False, "silu", True, True, False, None),
                 ("bf16", False, "relu", False, False, True, "z"), ("fp16", True, "none", True, True, True, None)]:
        with pinned(*kernel):
            plain.test_linear_backward(dev, cudair, M, N, K, *form)


@pytest.mark.parametrize("kernel", KERNELS, ids=NAMES)
@pytest.mark.parametrize("M,N,K", GRADIENT_SHAPES)
def test_gated_backward(dev, cudair, M, N, K, kernel):
    for form in [("bf16", True, "silu", False, False, False), ("fp16", False, "gelu_tanh", True, False, True),
                 ("bf16", False, "gelu", False, True, False)]:
        with pinned(*kernel):
            plain.test_gated_backward(dev, cudair, M, N, K, *form)


@pytest.mark.parametrize("kernel", KERNELS, ids=NAMES)
def test_calls_repeat_exactly(dev, cudair, kernel):
    """The same bits from a call however often and beside whatever it runs: no sum depends on timing."""
    import torch
    from cudair import kernels
    bf = torch.bfloat16
    gen = plain._gen(dev, 31)
    M, N, K = 1300, 2312, 1100
    x, dy, z = normal(gen, M, K, bf, dev), normal(gen, M, N, bf, dev), normal(gen, M, N, bf, dev)
    w = plain._weight(gen, N, K, bf, dev, True)
    new = lambda r, c: torch.empty(r, -(-c // 8) * 8, dtype=bf, device=dev)[:, :c]  # noqa: E731
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = [[new(M, N), new(M, N), new(M, K), new(N, K), torch.empty(N, device=dev)] for _ in streams]

    def run(o, s):
        kernels.linear(x, w, o[0], residual=z, act="gelu", b_trans=True, stream=s)
        kernels.linear_backward(dy, x, w, z=z, dz=o[1], da=o[2], db=o[3], dbias=o[4], act="silu", b_trans=True,
                                stream=s)

    with pinned(*kernel):
        run(outs[0], None)
        torch.cuda.synchronize()
        want = [t.clone() for t in outs[0]]
        for turn in range(8):
            for o, s in zip(outs, streams):
                for t in o:
                    t.fill_(7.0)
            torch.cuda.synchronize()
            for o, s in zip(outs, streams):
                run(o, s)
            torch.cuda.synchronize()
            for o in outs:
                assert all(torch.equal(t, v) for t, v in zip(o, want)), turn
    assert kernels.wait_status(clear=True) == 0


@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("last", ["linear", "linear_backward", "gated_backward"])
def test_weights_written_two_kernels_before(dev, cudair, mode, last):
    """A long kernel writes a matrix, a short one that needs nothing of it follows, and the third call's
    weights are that matrix: programmatic launches must not let the third read it before it is there.
    (Launch mode 2 lets a caller rule out the preceding kernel only.)"""
    import torch
    from cudair import kernels
    bf = torch.bfloat16
    n, K = 256, 1 << 18  # one tile, 4096 k-blocks: about a millisecond on two SMs
    a, b = (torch.randn(n, K, device=dev).to(bf) for _ in range(2))
    t, y = (torch.empty(n, n, dtype=bf, device=dev) for _ in range(2))
    s = torch.randn(n, n, device=dev).to(bf)
    one = torch.randn(8, n, device=dev).to(bf)
    z, dz, dg, du = (torch.randn(8, n, device=dev).to(bf) for _ in range(4))
    got = torch.empty(8, n, device=dev)

    def writer():
        kernels.set_linear_kernel(PAIRS, 256)
        kernels.linear(a, b, t, act="silu", b_trans=True)

    def between():
        kernels.linear(s, s, y)

    def reader():
        kernels.set_linear_kernel(SPLIT)
        if last == "linear":
            kernels.linear(one, t, got)
        elif last == "linear_backward":
            kernels.linear_backward(one, one, t, z=z, dz=dz, da=got, act="silu")
        else:
            kernels.gated_backward(one, one, t, t, z, z, dg, du, dx=got)

    try:
        writer()
        torch.cuda.synchronize()
        reader()
        torch.cuda.synchronize()
        want = got.clone()
        kernels.set_gemm_pdl(mode)
        for _ in range(10):
            t.fill_(11.0)
            got.fill_(0.0)
            torch.cuda.synchronize()
            writer()
            between()
            reader()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
    finally:
        kernels.set_gemm_pdl(0)
        kernels.set_linear_kernel(0)
    assert kernels.wait_status(clear=True) == 0


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("kernel", [(SPLIT, 0), (PAIRS, 0)], ids=["split", "pairs"])
@pytest.mark.parametrize("M,N,K", [(5, 264, 136), (1300, 2312, 1096)])
def test_captured_behind_copies_and_joins(dev, cudair, M, N, K, kernel, mode):
    """A capture in which calls follow a memset, a copy and the join of two streams, in each launch mode:
    replayed, the same bits as eagerly."""
    import torch
    from cudair import kernels
    bf = torch.bfloat16
    gen = plain._gen(dev, M, 51)
    rand = lambda r, c: torch.randn(r, c, generator=gen, device=dev).to(bf)  # noqa: E731
    x, src, w, dy, z = torch.empty(M, K, dtype=bf, device=dev), rand(M, K), rand(N, K), rand(M, N), rand(M, N)
    y, y2, dz, dy2 = (torch.empty(M, N, dtype=bf, device=dev) for _ in range(4))
    da, db, dbias = torch.empty_like(x), torch.empty_like(w), torch.empty(N, device=dev)
    outs, side = (y, y2, dz, da, db, dbias), torch.cuda.Stream()

    def run():
        main = torch.cuda.current_stream()
        x.zero_()
        x.copy_(src)
        kernels.linear(x, w, y, act="silu", b_trans=True)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            torch.mul(dy, 2, out=dy2)
            kernels.linear(x, w, y2, act="gelu", b_trans=True)
        main.wait_stream(side)
        kernels.linear_backward(dy2, x, w, z=z, dz=dz, da=da, db=db, dbias=dbias, act="silu", b_trans=True)

    kernels.set_gemm_pdl(mode)
    try:
        with pinned(*kernel):
            run()
            torch.cuda.synchronize()
            want = [t.clone() for t in outs]
            for t in outs:
                t.fill_(3.0)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                run()
            for _ in range(3):
                graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(t, v) for t, v in zip(outs, want))
    finally:
        kernels.set_gemm_pdl(0)
    assert kernels.wait_status(clear=True) == 0


def test_calls_from_several_threads(dev, cudair):
    """Four host threads, a stream each."""
    import threading

    import torch
    from cudair import kernels
    bf = torch.bfloat16
    x, w = torch.randn(200, 264, device=dev).to(bf), torch.randn(520, 264, device=dev).to(bf)
    want, outs, failed = torch.empty(200, 520, dtype=bf, device=dev), [], []
    kernels.linear(x, w, want, act="silu", b_trans=True)
    outs = [torch.empty_like(want) for _ in range(4)]
    torch.cuda.synchronize()

    def work(o):
        try:
            stream = torch.cuda.Stream()
            for _ in range(100):
                kernels.linear(x, w, o, act="silu", b_trans=True, stream=stream)
            stream.synchronize()
        except Exception as e:  # a thread's own failure is not raised by join
            failed.append(e)

    threads = [threading.Thread(target=work, args=(o,)) for o in outs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert all(torch.equal(o, want) for o in outs)
    assert kernels.wait_status(clear=True) == 0

"""What the entry points of the feed-forward operators launch, on CPU: the
object file of linear.cu linked with fakes of the kernels below it and of the
runtime's launch (linear_host/launches.cpp)."""
import itertools
import os
import re
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
PKG = os.path.join(os.path.dirname(HERE), "cuda-ir.go_b200")


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    """launches(call, modes, kernel, width) -> what the call's launches print."""
    sys.path.insert(0, PKG)
    import build
    build.build(force=False, verbose=False)
    exe = str(tmp_path_factory.mktemp("linear_host") / "launches")
    # nvcc finds its own headers and runtime; the host compiler alone may not.
    subprocess.run([build.NVCC, "-std=c++17", "-cudart", "shared", "-o", exe,
                    os.path.join(HERE, "linear_host", "launches.cpp"),
                    os.path.join(PKG, "_build", "linear.cu.o")], check=True, capture_output=True, text=True)

    def run(call, modes, kernel=0, width=0, refused=None):
        r = subprocess.run([exe, call] + [str(m) for m in modes] + ["--", str(kernel), str(width)],
                           capture_output=True, text=True, timeout=60)
        if refused:
            assert r.returncode == 1 and re.search(refused, r.stderr), (r.returncode, r.stderr)
            return []
        assert r.returncode == 0, (call, modes, r.returncode, r.stderr)
        return [{k: int(v) for k, v in re.findall(r"(\w+)=(\d+)", line)} | {"kernel": line.split()[0]}
                for line in r.stdout.splitlines()]
    return run


CALLS = {"linear": 1, "gated": 1, "linear_backward": 2, "gated_backward": 2}


@pytest.mark.parametrize("call", CALLS)
def test_launch_modes(launches, call):
    """Weights are requested early only where nothing that may still run writes them: behind the
    call's own element-wise kernel if that one waits for the stream, or if the caller says so."""
    for mode in (0, 1, 2):
        got = launches(call, [mode])
        assert len(got) == CALLS[call]
        product = got[-1]
        assert product["kernel"] == "product"
        assert product["programmatic"] == (1 if mode or len(got) == 2 else 0)
        assert product["weights_early"] == (1 if mode == 2 or (mode == 0 and len(got) == 2) else 0)
        if len(got) == 2:
            assert got[0]["kernel"] == "elementwise" and got[0]["programmatic"] == (1 if mode else 0)
            assert (got[0]["cluster"] > 0) == (call == "linear_backward")  # the bias's sums


@pytest.mark.parametrize("call", CALLS)
def test_a_mode_set_during_the_call_does_not_mix(launches, call):
    """Whatever the mode reads as during a call, its launches are those of one mode."""
    whole = [launches(call, [m]) for m in (0, 1, 2)]
    for modes in itertools.product((0, 1, 2), repeat=4):
        assert launches(call, modes) in whole, modes


@pytest.mark.parametrize("call", CALLS)
def test_the_kernel_may_be_chosen(launches, call):
    assert launches(call, [0], 1)[-1]["kernel"] == "product"  # the split kernel
    for width in (0, 192, 224, 256, 384, 448, 512):
        if call == "gated" and width in (224, 448):
            launches(call, [0], 2, width, refused="gated: tiles of %d columns do not take two weights" % width)
        else:
            got = launches(call, [0], 2, width)[-1]
            assert got["kernel"] == "pairs" and got["width"] == width


def test_kernel_choices_that_are_refused(cudair):
    from cudair import _lib, kernels
    for kernel, width, message in ((-1, 0, "linear kernel -1"), (3, 0, "linear kernel 3"), (2, 128, "tile width 128"),
                                   (2, -256, "tile width -256"), (1, 256, "tile width 256"), (0, 512, "tile width 512")):
        with pytest.raises(_lib.CudairError, match=message):
            kernels.set_linear_kernel(kernel, width)
    kernels.set_linear_kernel(0)


def test_depth_counts_both_contractions_of_dx(cudair):
    """dX = dG.Wg^T + dU.Wu^T is one sum over 2 N products."""
    import ctypes

    from cudair import _lib
    P = 0x7F0000000000
    n = 2 ** 25 + 8
    at = [P + (i << 40) for i in range(9)]
    args = dict(dh=at[0], x=None, wg=at[1], wu=at[2], g=at[3], u=at[4], dg=at[5], du=at[6], dx=at[7], M=4, N=n, K=16,
                lddh=n, ldwg=n, ldwu=n, ldg=n, ldu=n, lddg=n, lddu=n, lddx=16, act=4)
    assert cudair.lib().cudair_gated_backward(ctypes.byref(_lib.GatedBackwardArgs(**args)), None) == _lib.ERR_INVALID
    assert "contraction over 33554440 is too long (at most 33554432)" in cudair.last_error()
    # Without dX nothing sums over N: the next rule refuses this one.
    args.update(dx=None, x=at[5], ldx=16)
    assert cudair.lib().cudair_gated_backward(ctypes.byref(_lib.GatedBackwardArgs(**args)), None) == _lib.ERR_INVALID
    assert "dg lies over another matrix" in cudair.last_error()


# An output over part of another matrix of the call.  32 x 32 operands of 16 bits with a pitch of 64, so
# that the 32 other columns of a row are another matrix's; `at` and `ld` place one of them.
def _square(call, **over):
    from cudair import _lib
    P, n = 0x7F0000000000, 32
    names = {"cudair_linear": (_lib.LinearArgs, "a b residual d z", "bias"),
             "cudair_linear_backward": (_lib.LinearBackwardArgs, "dy a b z dz da db", "dbias"),
             "cudair_gated": (_lib.GatedArgs, "x wg wu h g u", None),
             "cudair_gated_backward": (_lib.GatedBackwardArgs, "dh x wg wu g u dg du dx dwg dwu", None)}[call]
    cls, mats, vector = names
    args = dict(M=n, N=n, K=n, act=4)
    for i, m in enumerate(mats.split()):
        args[m], args["ld" + {"residual": "res"}.get(m, m)] = P + (i << 20), 64
    if vector:
        args[vector] = P + (100 << 20)
    args.update(over)
    return cls(**args)


def _refused(cudair, call, **over):
    import ctypes

    from cudair import _lib
    args = _square(call, **over)
    rc = getattr(cudair.lib(), call)(ctypes.byref(args), None)
    assert rc == _lib.ERR_INVALID, (rc, cudair.last_error())
    return cudair.last_error()


AT = 0x7F0000000000
PARTIAL = [  # call, output, what it lies over, that one's place in the order of _square
    ("cudair_linear", "d", "a", 0), ("cudair_linear", "d", "b", 1), ("cudair_linear", "d", "residual", 2),
    ("cudair_linear", "z", "d", 3), ("cudair_linear", "z", "residual", 2),
    ("cudair_gated", "h", "x", 0), ("cudair_gated", "g", "wu", 2), ("cudair_gated", "u", "g", 4),
    ("cudair_linear_backward", "dz", "dy", 0), ("cudair_linear_backward", "dz", "z", 3),
    ("cudair_linear_backward", "da", "a", 1), ("cudair_linear_backward", "db", "da", 5),
    ("cudair_gated_backward", "dg", "g", 4), ("cudair_gated_backward", "du", "dh", 0),
    ("cudair_gated_backward", "du", "dg", 6), ("cudair_gated_backward", "dx", "u", 5),
    ("cudair_gated_backward", "dwu", "dwg", 9)]


@pytest.mark.parametrize("call,out,other,place", PARTIAL)
def test_partial_overlaps_are_refused(cudair, call, out, other, place):
    base = AT + (place << 20)
    for shift in (16, 48, 128, 31 * 128 + 48, -16, -48, -31 * 128):
        assert re.search("lies over another matrix|share memory", _refused(cudair, call, **{out: base + shift})), shift
    # Another pitch: rows of 80 elements run into the other's columns.
    assert re.search("lies over another matrix|share memory|pitch",
                     _refused(cudair, call, **{out: base - 64, "ld" + out: 80}))


def test_vectors_that_overlap_are_refused(cudair):
    for at in (AT + (3 << 20) + 60, AT + (3 << 20) - 64, AT + (3 << 20) + 31 * 128 + 60):
        assert "d lies over another" in _refused(cudair, "cudair_linear", bias=at)
    for place in (0, 1, 2, 3, 4, 5, 6):
        assert "dbias lies over another" in _refused(cudair, "cudair_linear_backward", dbias=AT + (place << 20) - 4)


def test_matrices_side_by_side_are_not_refused(launches, cudair):
    """Columns of one array beside one another, and one after the other: accepted up to the launch."""
    import ctypes

    from cudair import _lib
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are not real")
    for call, out, other, place in PARTIAL:
        base = AT + (place << 20)
        for shift in (64, -64, 32 * 128, -32 * 128, 32 * 128 - 64):
            rc = getattr(cudair.lib(), call)(ctypes.byref(_square(call, **{out: base + shift})), None)
            assert rc != _lib.ERR_INVALID, (call, out, other, shift, cudair.last_error())


def test_overlap_is_exact(cudair):
    """d and z of random pitches, types and distances: refused if and only if they have a byte in common."""
    import ctypes
    import random

    from cudair import _lib
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are not real")

    def spans(at, pitch, row, rows):
        return {at + i * pitch + j for i in range(rows) for j in range(0, row, 2)}

    rng, seen = random.Random(7), [0, 0]
    for _ in range(2500):
        M, N, f32 = rng.choice([1, 1, 2, 3, 7]), rng.choice([1, 3, 8, 20]), rng.random() < 0.5
        ldd, ldz = (-(-N // 8) * 8 + 8 * rng.randrange(6) for _ in range(2))
        d, z = AT + (1 << 20), AT + (1 << 20) + 16 * rng.randrange(-30, 30)
        args = _lib.LinearArgs(a=AT, b=AT + (8 << 20), d=d, z=z, M=M, N=N, K=8, lda=8, ldb=24, ldd=ldd, ldz=ldz,
                               flags=0x10 if f32 else 0)
        rc = cudair.lib().cudair_linear(ctypes.byref(args), None)
        want = bool(spans(d, ldd * (4 if f32 else 2), N * (4 if f32 else 2), M) & spans(z, ldz * 2, N * 2, M))
        assert (rc == _lib.ERR_INVALID) == want, (M, N, f32, ldd, ldz, z - d, cudair.last_error())
        seen[want] += 1
    assert min(seen) > 300


def test_pitches_of_operands_that_are_not_needed(cudair):
    """Without db nothing reads a: its pitch is not looked at, and only its first row is kept clear of."""
    import ctypes

    from cudair import _lib
    import torch
    if torch.cuda.is_available():
        pytest.skip("the addresses are not real")
    for ld in (0, -8, 7, 2 ** 29 + 8, 2 ** 61 + 3, 2 ** 63 - 1):
        args = _square("cudair_linear_backward", db=None, lda=ld)
        assert cudair.lib().cudair_linear_backward(ctypes.byref(args), None) != _lib.ERR_INVALID, (ld, cudair.last_error())
        assert "da lies over another" in _refused(cudair, "cudair_linear_backward", db=None, lda=ld,
                                                  da=AT + (1 << 20) + 48)

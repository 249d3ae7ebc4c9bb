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

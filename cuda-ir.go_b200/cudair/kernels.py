"""Launchers of the tuned sm_100a kernels over the C ABI, taking torch CUDA
tensors (device memory and streams come from torch; the arithmetic is the
library's).  Each call is asynchronous on the given stream (default: torch's
current stream).
"""
from __future__ import annotations

import ctypes

from ._lib import (CudairError, GatedArgs, GatedBackwardArgs, LinearArgs, LinearBackwardArgs, check, lib)


def _stream(stream):
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _need(t, dtype, name):
    import torch
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise CudairError(1, f"cudair: {name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise CudairError(1, f"cudair: {name} must be {dtype}, got {t.dtype}")
    # The library launches on the current device; a tensor of another GPU
    # would be read across NVLink by the kernels (or fail to launch).
    cur = torch.cuda.current_device()
    if t.device.index != cur:
        raise CudairError(1, f"cudair: {name} is on {t.device}, the current device is cuda:{cur}")


def matmul16(a, b, c, stream=None) -> None:
    """c += a @ b for n x n row-major fp16 a, b and fp32 c (MatMul16's operands)."""
    import torch
    _need(a, torch.float16, "a")
    _need(b, torch.float16, "b")
    _need(c, torch.float32, "c")
    n = a.shape[0]
    if not (a.shape == b.shape == c.shape == (n, n)) or not (
            a.is_contiguous() and b.is_contiguous() and c.is_contiguous()):
        raise CudairError(1, "cudair: MatMul16: a, b, c must be contiguous n x n")
    check(lib().cudair_matmul16(a.data_ptr(), b.data_ptr(), c.data_ptr(), n, _stream(stream)))


def gemm(a, b, c, stream=None) -> None:
    """c += a @ b: a (M x K) and b (K x N) fp16, c (M x N) fp32, row-major with
    unit inner stride."""
    import torch
    _need(a, torch.float16, "a")
    _need(b, torch.float16, "b")
    _need(c, torch.float32, "c")
    M, K = a.shape
    K2, N = b.shape
    if K2 != K or tuple(c.shape) != (M, N):
        raise CudairError(1, f"cudair: gemm: shapes {tuple(a.shape)} {tuple(b.shape)} {tuple(c.shape)}")
    for t, nm in ((a, "a"), (b, "b"), (c, "c")):
        if t.stride(1) != 1:
            raise CudairError(1, f"cudair: gemm: {nm} needs unit inner stride")
    check(lib().cudair_gemm_f16f32(a.data_ptr(), b.data_ptr(), c.data_ptr(), M, N, K,
                                   a.stride(0), b.stride(0), c.stride(0), _stream(stream)))


GEMM_BF16, GEMM_B_T, GEMM_OVERWRITE, GEMM_C_F16 = 0x1, 0x2, 0x4, 0x8


def gemm_ex(a, b, c, bias=None, b_trans=False, overwrite=False, stream=None) -> None:
    """The tensor-package GEMM family on the tcgen05 kernels (cudair_gemm):
    c (+)= a @ B with B = b, or b.T when b_trans (b is N x K).  a and b are
    both fp16 or both bf16; c is fp32 (accumulated into, or written when
    overwrite) or fp16 (written: needs overwrite); bias (fp32 M x N) gives
    c = a @ B + bias."""
    import torch
    if a.dtype not in (torch.float16, torch.bfloat16) or b.dtype != a.dtype:
        raise CudairError(1, "cudair: gemm_ex: a and b must be both float16 or both bfloat16")
    for t, nm in ((a, "a"), (b, "b"), (c, "c")):
        _need(t, t.dtype, nm)
        if t.stride(1) != 1:
            raise CudairError(1, f"cudair: gemm_ex: {nm} needs unit inner stride")
    if c.dtype not in (torch.float32, torch.float16):
        raise CudairError(1, "cudair: gemm_ex: c must be float32 or float16")
    M, K = a.shape
    N = b.shape[0] if b_trans else b.shape[1]
    if (b.shape[1] if b_trans else b.shape[0]) != K or tuple(c.shape) != (M, N):
        raise CudairError(1, f"cudair: gemm_ex: shapes {tuple(a.shape)} {tuple(b.shape)} {tuple(c.shape)}")
    flags = (GEMM_BF16 if a.dtype == torch.bfloat16 else 0) | (GEMM_B_T if b_trans else 0) | \
        (GEMM_OVERWRITE if overwrite else 0) | (GEMM_C_F16 if c.dtype == torch.float16 else 0)
    bias_ptr, ldbias = None, 0
    if bias is not None:
        _need(bias, torch.float32, "bias")
        if tuple(bias.shape) != (M, N) or bias.stride(1) != 1:
            raise CudairError(1, "cudair: gemm_ex: bias must be M x N with unit inner stride")
        bias_ptr, ldbias = bias.data_ptr(), bias.stride(0)
    check(lib().cudair_gemm(a.data_ptr(), b.data_ptr(), c.data_ptr(), bias_ptr, M, N, K, a.stride(0),
                            b.stride(0), c.stride(0), ldbias, flags, _stream(stream)))


ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
LINEAR_D_F32, LINEAR_BIAS_16, LINEAR_DA_F32, LINEAR_DB_F32 = 0x10, 0x20, 0x40, 0x80


def _act(op, act):
    try:
        return ACTIVATIONS[act]
    except (KeyError, TypeError):
        raise CudairError(1, f"cudair: {op}: act must be one of {', '.join(ACTIVATIONS)}, got {act!r}") from None


def _type(op, t, name):
    """The 16-bit type of an operation's operands, from its first one."""
    import torch
    dt = getattr(t, "dtype", None)
    if dt is not torch.float16 and dt is not torch.bfloat16:
        raise CudairError(1, f"cudair: {op}: {name} must be a float16 or bfloat16 tensor, got {dt}")
    return dt


def _mat(op, name, t, dtypes, rows, cols, device):
    """Checks a rows x cols matrix and returns its pointer and row pitch."""
    if not getattr(t, "is_cuda", False):
        raise CudairError(1, f"cudair: {op}: {name} must be a CUDA tensor")
    if t.dtype not in dtypes:
        raise CudairError(1, f"cudair: {op}: {name} must be {' or '.join(map(str, dtypes))}, got {t.dtype}")
    if t.get_device() != device:
        raise CudairError(1, f"cudair: {op}: {name} is on {t.device}, the current device is cuda:{device}")
    if t.shape != (rows, cols):
        raise CudairError(1, f"cudair: {op}: {name} must be {rows} x {cols}, got {tuple(t.shape)}")
    ld, inner = t.stride()
    if inner != 1 and cols > 1:
        raise CudairError(1, f"cudair: {op}: {name} needs unit inner stride")
    # One row has no pitch of its own, and an empty matrix no rows.
    return t.data_ptr(), -(-cols // 8) * 8 if rows <= 1 or cols == 0 else ld


def _device():
    import torch
    return torch.cuda.current_device()


def _current_stream(stream, device):
    """_stream without building a torch Stream object (3 us)."""
    if stream is None:
        import torch
        return torch._C._cuda_getCurrentRawStream(device)
    return _stream(stream)


def _dims(op, x, xname, w, wname, b_trans):
    """(M, N, K) of x (M x K) and a weight (K x N, or N x K with b_trans)."""
    if getattr(x, "ndim", 0) != 2 or getattr(w, "ndim", 0) != 2:
        raise CudairError(1, f"cudair: {op}: {xname} and {wname} must be matrices")
    return x.shape[0], w.shape[0 if b_trans else 1], x.shape[1]


def _grad_dims(op, dy, yname, x, w, dx, dw, b_trans):
    """(M, N, K) of a gradient's call: M x N from the upstream gradient, K from the
    first of x, w, dx and dw that is given (0: none, and no product to compute)."""
    for t, name in ((dy, yname), (x, "the input"), (w, "the weight"), (dx, "the input's gradient"),
                    (dw, "the weight's gradient")):
        if (t is not None or t is dy) and getattr(t, "ndim", 0) != 2:
            raise CudairError(1, f"cudair: {op}: {name} must be a matrix")
    for t, dim in ((x, 1), (w, 1 if b_trans else 0), (dx, 1), (dw, 1 if b_trans else 0)):
        if t is not None:
            return dy.shape[0], dy.shape[1], t.shape[dim]
    return dy.shape[0], dy.shape[1], 0


def _optional(op, name, t, dtypes, rows, cols, device):
    return (None, 0) if t is None else _mat(op, name, t, dtypes, rows, cols, device)


def linear(a, b, d, bias=None, residual=None, z=None, act="none", b_trans=False, stream=None) -> None:
    """d = act(a @ B + bias) + residual with B = b (K x N), or b.T when b_trans
    (b is N x K): one kernel (cudair_linear).  a and b are both fp16 or both
    bf16; d is of their type or fp32; bias has N values (fp32 or a's type);
    residual is M x N of d's type and may be d itself; z (M x N of a's type)
    receives a @ B + bias for linear_backward.  act: "none", "relu", "gelu",
    "gelu_tanh" or "silu".  Rows start on 16 bytes."""
    import torch
    op, dev = "linear", _device()
    dt = _type(op, a, "a")
    M, N, K = _dims(op, a, "a", b, "b", b_trans)
    t16, flags = (dt,), (GEMM_BF16 if dt is torch.bfloat16 else 0) | (GEMM_B_T if b_trans else 0)
    pa, lda = _mat(op, "a", a, t16, M, K, dev)
    pb, ldb = _mat(op, "b", b, t16, N if b_trans else K, K if b_trans else N, dev)
    pd, ldd = _mat(op, "d", d, (dt, torch.float32), M, N, dev)
    if d.dtype is torch.float32:
        flags |= LINEAR_D_F32
    pbias, pres, ldres, pz, ldz = None, None, 0, None, 0
    if bias is not None:
        if bias.shape != (N,) or (N > 1 and bias.stride(0) != 1):
            raise CudairError(1, f"cudair: {op}: bias must have {N} consecutive values")
        pbias = _mat(op, "bias", bias.view(1, N), (torch.float32, dt), 1, N, dev)[0]
        if bias.dtype is not torch.float32:
            flags |= LINEAR_BIAS_16
    if residual is not None:
        pres, ldres = _mat(op, "residual", residual, (d.dtype,), M, N, dev)
    if z is not None:
        pz, ldz = _mat(op, "z", z, t16, M, N, dev)
    check(lib().cudair_linear(ctypes.byref(LinearArgs(
        pa, pb, pbias, pres, pd, pz, M, N, K, lda, ldb, ldres, ldd, ldz, _act(op, act), flags)),
        _current_stream(stream, dev)))


def linear_backward(dy, a, b, z=None, dz=None, da=None, db=None, dbias=None, act="none", b_trans=False,
                    stream=None) -> None:
    """The gradients of linear (cudair_linear_backward), each written where
    given: da = dz @ B.T (M x K), db = a.T @ dz (stored as b is), dbias (N
    fp32 values) = dz summed over its rows, with dz = dy * act'(z).  dy is of
    a's type or fp32 (the gradient of d, and so the residual's).  z (as linear
    stored it) is needed with an activation; dz (M x N of a's type) with an
    activation or an fp32 dy, and only then; it may be z's or dy's memory.
    da and db are of a's type or fp32.  a may be None without db (a frozen
    weight), b without da."""
    import torch
    op, dev = "linear_backward", _device()
    typed, name = next(((t, n) for t, n in ((a, "a"), (b, "b"), (dz, "dz"), (z, "z")) if t is not None), (dy, "dy"))
    dt = _type(op, typed, name)
    M, N, K = _grad_dims(op, dy, "dy", a, b, da, db, b_trans)
    t16, either = (dt,), (dt, torch.float32)
    w = (N, K) if b_trans else (K, N)
    flags = (GEMM_BF16 if dt is torch.bfloat16 else 0) | (GEMM_B_T if b_trans else 0)
    pdy, lddy = _mat(op, "dy", dy, either, M, N, dev)
    if dy.dtype is torch.float32:
        flags |= LINEAR_D_F32
    pa, lda = _optional(op, "a", a, t16, M, K, dev)
    pb, ldb = _optional(op, "b", b, t16, *w, dev)
    pz = pdz = pda = pdb = pdbias = None
    ldz = lddz = ldda = lddb = 0
    if z is not None:
        pz, ldz = _mat(op, "z", z, t16, M, N, dev)
    if dz is not None:
        pdz, lddz = _mat(op, "dz", dz, t16, M, N, dev)
    if da is not None:
        pda, ldda = _mat(op, "da", da, either, M, K, dev)
        flags |= LINEAR_DA_F32 if da.dtype is torch.float32 else 0
    if db is not None:
        pdb, lddb = _mat(op, "db", db, either, *w, dev)
        flags |= LINEAR_DB_F32 if db.dtype is torch.float32 else 0
    if dbias is not None:
        if dbias.shape != (N,) or (N > 1 and dbias.stride(0) != 1):
            raise CudairError(1, f"cudair: {op}: dbias must have {N} consecutive values")
        pdbias = _mat(op, "dbias", dbias.view(1, N), (torch.float32,), 1, N, dev)[0]
    check(lib().cudair_linear_backward(ctypes.byref(LinearBackwardArgs(
        pdy, pa, pb, pz, pdz, pda, pdb, pdbias, M, N, K, lddy, lda, ldb, ldz, lddz, ldda, lddb, _act(op, act),
        flags)), _current_stream(stream, dev)))


def gated(x, wg, wu, h, g=None, u=None, act="silu", b_trans=False, stream=None) -> None:
    """h = act(x @ Wg) * (x @ Wu) in one kernel (cudair_gated), with Wg = wg
    and Wu = wu (K x N), or their transposes when b_trans (both N x K).  All
    fp16 or all bf16; g and u (both or neither, M x N) receive the two products for
    gated_backward.  The weights may be halves of one tensor."""
    import torch
    op, dev = "gated", _device()
    dt = _type(op, x, "x")
    M, N, K = _dims(op, x, "x", wg, "wg", b_trans)
    t16 = (dt,)
    w = (N, K) if b_trans else (K, N)
    flags = (GEMM_BF16 if dt is torch.bfloat16 else 0) | (GEMM_B_T if b_trans else 0)
    px, ldx = _mat(op, "x", x, t16, M, K, dev)
    pwg, ldwg = _mat(op, "wg", wg, t16, *w, dev)
    pwu, ldwu = _mat(op, "wu", wu, t16, *w, dev)
    ph, ldh = _mat(op, "h", h, t16, M, N, dev)
    pg, ldg = (None, 0) if g is None else _mat(op, "g", g, t16, M, N, dev)
    pu, ldu = (None, 0) if u is None else _mat(op, "u", u, t16, M, N, dev)
    check(lib().cudair_gated(ctypes.byref(GatedArgs(
        px, pwg, pwu, ph, pg, pu, M, N, K, ldx, ldwg, ldwu, ldh, ldg, ldu, _act(op, act), flags)),
        _current_stream(stream, dev)))


def gated_backward(dh, x, wg, wu, g, u, dg, du, dx=None, dwg=None, dwu=None, act="silu", b_trans=False,
                   stream=None) -> None:
    """The gradients of gated (cudair_gated_backward): dg = dh * u * act'(g)
    and du = dh * act(g) (M x N; they may be g's and u's memory), then, where
    given, dx = dg @ Wg.T + du @ Wu.T and dwg = x.T @ dg, dwu = x.T @ du
    (stored as the weights are; both or neither).  dx and the weights'
    gradients are of dh's type or fp32.  x may be None without dwg and dwu
    (frozen weights), wg and wu without dx."""
    import torch
    op, dev = "gated_backward", _device()
    dt = _type(op, dh, "dh")
    M, N, K = _grad_dims(op, dh, "dh", x, wg, dx, dwg, b_trans)
    t16, either = (dt,), (dt, torch.float32)
    w = (N, K) if b_trans else (K, N)
    flags = (GEMM_BF16 if dt is torch.bfloat16 else 0) | (GEMM_B_T if b_trans else 0)
    pdh, lddh = _mat(op, "dh", dh, t16, M, N, dev)
    px, ldx = _optional(op, "x", x, t16, M, K, dev)
    pwg, ldwg = _optional(op, "wg", wg, t16, *w, dev)
    pwu, ldwu = _optional(op, "wu", wu, t16, *w, dev)
    pg, ldg = _mat(op, "g", g, t16, M, N, dev)
    pu, ldu = _mat(op, "u", u, t16, M, N, dev)
    pdg, lddg = _mat(op, "dg", dg, t16, M, N, dev)
    pdu, lddu = _mat(op, "du", du, t16, M, N, dev)
    pdx = pdwg = pdwu = None
    lddx = lddwg = lddwu = 0
    if dx is not None:
        pdx, lddx = _mat(op, "dx", dx, either, M, K, dev)
        flags |= LINEAR_DA_F32 if dx.dtype is torch.float32 else 0
    if dwg is not None:
        pdwg, lddwg = _mat(op, "dwg", dwg, either, *w, dev)
        flags |= LINEAR_DB_F32 if dwg.dtype is torch.float32 else 0
    if dwu is not None:
        pdwu, lddwu = _mat(op, "dwu", dwu, (dwg.dtype,) if dwg is not None else either, *w, dev)
    check(lib().cudair_gated_backward(ctypes.byref(GatedBackwardArgs(
        pdh, px, pwg, pwu, pg, pu, pdg, pdu, pdx, pdwg, pdwu, M, N, K, lddh, ldx, ldwg, ldwu, ldg, ldu, lddg,
        lddu, lddx, lddwg, lddwu, _act(op, act), flags)), _current_stream(stream, dev)))


def gemm_host(a_h, b_h, c_h, a_d, b_d, c_d, rows_per_block=0, stream=None) -> None:
    """c_h += a_h @ b_h from host (CPU) tensors, through the caller's device
    buffers a_d, b_d, c_d (dense, same shapes): copies in, GEMM and copy out
    pipelined over tiles of C (rows_per_block > 0: full-width row blocks of
    that height; 0: automatic).  b_h = None: b_d already holds B.
    Asynchronous on `stream`; c_h holds the result once the stream is
    synchronised.  Pinned host tensors let the copies overlap."""
    import torch
    for t, dt, nm in ((a_h, torch.float16, "a_h"), (b_h, torch.float16, "b_h"),
                      (c_h, torch.float32, "c_h")):
        if t is None and nm == "b_h":
            continue  # B already in b_d
        if not isinstance(t, torch.Tensor) or t.is_cuda or t.dtype != dt or t.stride(1) != 1:
            raise CudairError(1, f"cudair: gemm_host: {nm} must be a host {dt} tensor, unit inner stride")
    for t, dt, nm in ((a_d, torch.float16, "a_d"), (b_d, torch.float16, "b_d"),
                      (c_d, torch.float32, "c_d")):
        _need(t, dt, nm)
        if not t.is_contiguous():
            raise CudairError(1, f"cudair: gemm_host: {nm} must be contiguous")
    M, K = a_h.shape
    K2, N = b_d.shape
    if K2 != K or tuple(c_h.shape) != (M, N) or tuple(a_d.shape) != (M, K) or \
            tuple(c_d.shape) != (M, N) or (b_h is not None and tuple(b_h.shape) != (K, N)):
        raise CudairError(1, "cudair: gemm_host: shapes do not match")
    check(lib().cudair_gemm_f16f32_host(
        a_h.data_ptr(), None if b_h is None else b_h.data_ptr(), c_h.data_ptr(), M, N, K,
        a_h.stride(0), N if b_h is None else b_h.stride(0),
        c_h.stride(0), a_d.data_ptr(), b_d.data_ptr(), c_d.data_ptr(), rows_per_block,
        _stream(stream)))


def _host_tensor(t, dtype, name):
    import torch
    if not isinstance(t, torch.Tensor) or t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise CudairError(1, f"cudair: {name} must be a contiguous host {dtype} tensor")


def vecadd_host(a_h, b_h, out_h, a_d, b_d, out_d, chunk=0, stream=None) -> None:
    """out_h = a_h + b_h from host (CPU) fp32 vectors through the caller's
    device buffers (cudair_vecadd_host): copies in, VecAdd and copies out
    pipelined over chunks.  Asynchronous on `stream`; pinned host tensors let
    the copies overlap."""
    import torch
    for t, nm in ((a_h, "a_h"), (b_h, "b_h"), (out_h, "out_h")):
        _host_tensor(t, torch.float32, nm)
    for t, nm in ((a_d, "a_d"), (b_d, "b_d"), (out_d, "out_d")):
        _need(t, torch.float32, nm)
    n = out_h.numel()
    if any(t.numel() != n for t in (a_h, b_h, a_d, b_d, out_d)):
        raise CudairError(1, "cudair: vecadd_host: length mismatch")
    check(lib().cudair_vecadd_host(a_h.data_ptr(), b_h.data_ptr(), out_h.data_ptr(), n, a_d.data_ptr(),
                                   b_d.data_ptr(), out_d.data_ptr(), chunk, _stream(stream)))


def matmul16_host(a_h, b_h, c_h, a_d, b_d, c_d, stream=None) -> None:
    """c_h += a_h @ b_h for n x n host tensors (MatMul16's operands) through
    the caller's device buffers (cudair_matmul16_host).  Asynchronous on
    `stream`."""
    import torch
    _host_tensor(a_h, torch.float16, "a_h")
    _host_tensor(b_h, torch.float16, "b_h")
    _host_tensor(c_h, torch.float32, "c_h")
    _need(a_d, torch.float16, "a_d")
    _need(b_d, torch.float16, "b_d")
    _need(c_d, torch.float32, "c_d")
    n = c_h.shape[0]
    if any(tuple(t.shape) != (n, n) for t in (a_h, b_h, c_h, a_d, b_d, c_d)):
        raise CudairError(1, "cudair: matmul16_host: every operand must be n x n")
    check(lib().cudair_matmul16_host(a_h.data_ptr(), b_h.data_ptr(), c_h.data_ptr(), n, a_d.data_ptr(),
                                     b_d.data_ptr(), c_d.data_ptr(), _stream(stream)))


def set_gemm_variant(variant: int) -> None:
    """0 = automatic, 1 = single-CTA 128x256 tiles, 2 = CTA-pair 256x256 tiles,
    3 = few-row kernel (M <= 128), 4 = CTA-pair 256x512 tiles, 5 = small-problem
    kernel (K <= 512), 6 = few-row kernel with k-chunks handed out at run time
    (M <= 64)."""
    check(lib().cudair_set_gemm_variant(variant))


def set_gemm_pdl(mode: int) -> None:
    """Programmatic dependent launch of the few-row GEMM: 0 off, 1 on, 2 on
    with B (weights, not written by the preceding kernel) requested early."""
    check(lib().cudair_set_gemm_pdl(mode))


def set_linear_kernel(kernel: int, width: int = 0) -> None:
    """The kernel of linear, gated and their gradients: 0 = automatic, 1 = split
    kernel, 2 = CTA pairs with tiles of width 192, 224, 256, 384, 448 or 512
    (gated: not 224 or 448) or, with 0, the automatic one."""
    check(lib().cudair_set_linear_kernel(kernel, width))


def vecadd(a, b, out, stream=None) -> None:
    """out = a + b over fp32 vectors (VecAdd's operands)."""
    import torch
    for t, nm in ((a, "a"), (b, "b"), (out, "out")):
        _need(t, torch.float32, nm)
    n = out.numel()
    if a.numel() != n or b.numel() != n:
        raise CudairError(1, "cudair: VecAdd: length mismatch")
    check(lib().cudair_vecadd(a.data_ptr(), b.data_ptr(), out.data_ptr(), n, _stream(stream)))


def saxpy(alpha, x, y, stream=None) -> None:
    """y = alpha * x + y over fp32 vectors (Saxpy's operands)."""
    import torch
    _need(x, torch.float32, "x")
    _need(y, torch.float32, "y")
    if x.numel() != y.numel():
        raise CudairError(1, "cudair: Saxpy: length mismatch")
    check(lib().cudair_saxpy(float(alpha), x.data_ptr(), y.data_ptr(), y.numel(), _stream(stream)))


def square(x, stream=None) -> None:
    """x = x * x in place over an fp32 vector (Square's operand)."""
    import torch
    _need(x, torch.float32, "x")
    check(lib().cudair_square(x.data_ptr(), x.numel(), _stream(stream)))


def reduce_f32(x, out, stream=None) -> None:
    """out[2w], out[2w+1] = min, max of warp w's 32 values (ReduceF32)."""
    import torch
    _need(x, torch.float32, "in")
    _need(out, torch.float32, "out")
    check(lib().cudair_reduce_f32(x.data_ptr(), out.data_ptr(), x.numel(), _stream(stream)))


FILL_F32, FILL_F16 = 0, 1
FILL_UNIFORM, FILL_NORMAL = 0, 1


def _fill(t, dist, seed, p0, p1, offset, stream):
    import torch
    if t.dtype not in (torch.float32, torch.float16):
        raise CudairError(1, f"cudair: fill: tensor must be float32 or float16, got {t.dtype}")
    _need(t, t.dtype, "out")
    if not t.is_contiguous():
        raise CudairError(1, "cudair: fill: tensor must be contiguous")
    check(lib().cudair_fill(t.data_ptr(), FILL_F16 if t.dtype == torch.float16 else FILL_F32, dist,
                            t.numel(), seed, offset, float(p0), float(p1), _stream(stream)))


def fill_uniform(t, seed: int, lo=-1.0, hi=1.0, offset: int = 0, stream=None) -> None:
    """Fills t (contiguous fp32 or fp16) with elements offset.. of the seeded
    U(lo, hi) stream (cudair_fill), bit for bit the CPU oracle's values."""
    _fill(t, FILL_UNIFORM, seed, lo, hi, offset, stream)


def fill_normal(t, seed: int, mean=0.0, std=1.0, offset: int = 0, stream=None) -> None:
    """Fills t (contiguous fp32 or fp16) with elements offset.. of the seeded
    N(mean, std) stream (cudair_fill), bit for bit the CPU oracle's values."""
    _fill(t, FILL_NORMAL, seed, mean, std, offset, stream)


def wait_status(clear: bool = True) -> int:
    """Synchronises and returns the bounded-wait status word (0 = no wait gave
    up); raises CudairError(ERR_TIMEOUT) when a bit is set."""
    v = ctypes.c_uint32()
    rc = lib().cudair_wait_status(ctypes.byref(v), 1 if clear else 0)
    if rc != 0:
        err = CudairError(rc, lib().cudair_last_error().decode())
        err.status = v.value
        raise err
    return v.value


def wait_timeout_selftest(limit_ns: int, stream=None) -> None:
    check(lib().cudair_wait_timeout_selftest(limit_ns, _stream(stream)))

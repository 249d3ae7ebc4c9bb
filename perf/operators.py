"""What the feed-forward operators cost: the matrix product with bias,
activation and residual in its epilogue (`linear`), the gated projection
(`gated`), and the backward pass of each, in cases over the range a program
that serves or trains a transformer calls them with.

`run` computes a case in its plain form (elementary torch operations in
32 bits, rounded once at the end) while `own` is false, and through
cudair.kernels while it is true.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

# Cases.  M tokens, K inputs, N (or F) outputs.  "rows": weights stored one
# row per output (N x K, as a checkpoint has them), else one row per input
# (K x N, the layout MatMul16 and the decode GEMM read).  Row pitches are the
# widths rounded up to eight elements.
_LISTED = [
    # The latency end: one token through an output projection, added to the
    # residual stream, as in every layer of every decode step.
    dict(name="linear token", op="linear", M=1, N=4096, K=4096, dtype="bf16", rows=True, act="none",
         bias=False, residual=True, save=False),
    # Sixteen sequences decoded together, the decode GEMM's own shape.
    dict(name="linear decode 16", op="linear", M=16, N=14336, K=4096, dtype="fp16", rows=False,
         act="gelu_tanh", bias=True, residual=False, save=False),
    # A ragged training batch through an odd-sized layer; the
    # pre-activation is kept for the backward pass.
    dict(name="linear ragged", op="linear", M=777, N=1003, K=519, dtype="bf16", rows=True, act="gelu",
         bias=True, residual=True, save=True),
    # The largest forward product: a long prompt through a square layer.
    dict(name="linear 8192", op="linear", M=8192, N=8192, K=8192, dtype="fp16", rows=False, act="relu",
         bias=True, residual=True, save=False),
    # A training step of the same kind of layer, and an odd one.
    dict(name="linear backward", op="linear_backward", M=4096, N=14336, K=4096, dtype="bf16", rows=False,
         act="gelu_tanh", bias=True),
    dict(name="linear backward ragged", op="linear_backward", M=301, N=515, K=1029, dtype="fp16", rows=True,
         act="relu", bias=True),
    # A decode step's gated projection: one token, and a batch of 64.
    dict(name="gated token", op="gated", M=1, N=14336, K=4096, dtype="bf16", rows=True, act="silu",
         save=False),
    dict(name="gated decode 64", op="gated", M=64, N=14336, K=4096, dtype="fp16", rows=False, act="silu",
         save=False),
    # The forward pass of a training step (gate and up are kept), and an
    # odd one.
    dict(name="gated prompt", op="gated", M=4096, N=14336, K=4096, dtype="bf16", rows=True, act="silu",
         save=True),
    dict(name="gated ragged", op="gated", M=333, N=1357, K=1091, dtype="fp16", rows=False,
         act="gelu_tanh", save=True),
    # The backward pass of the two.
    dict(name="gated backward", op="gated_backward", M=4096, N=14336, K=4096, dtype="bf16", rows=True,
         act="silu"),
    dict(name="gated backward ragged", op="gated_backward", M=203, N=1731, K=777, dtype="bf16",
         rows=False, act="gelu"),
]


def listed():
    return [dict(c) for c in _LISTED]


def _spread(rng, lo, hi):
    """A size between lo and hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_backward", "gated", "gated", "gated_backward"])
    case = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), rows=rng.random() < 0.5)
    training = op.endswith("backward")
    while True:
        M = _spread(rng, 1, 128) if not training and rng.random() < 0.5 else _spread(rng, 16, 8192)
        N, K = _spread(rng, 96, 14336), _spread(rng, 64, 8192)
        if rng.random() < 0.5:  # widths of real layers are mostly whole multiples
            N, K = -(-N // 128) * 128, -(-K // 128) * 128
        case.update(M=M, N=N, K=K)
        if work(case)["flops"] <= 1.0e12:
            break
    if op.startswith("linear"):
        case["act"] = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
        case["bias"] = rng.random() < 0.5
    else:
        case["act"] = rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"])
    if op == "linear":
        case["residual"] = rng.random() < 0.5
    if not training:
        case["save"] = M > 128 and case["act"] != "none" and rng.random() < 0.5
    return case


def work(case):
    """Bytes and operations of one pass: each input once, each output once."""
    M, N, K = case["M"], case["N"], case["K"]
    op = case["op"]
    x, w, y = 2 * M * K, 2 * N * K, 2 * M * N
    if op == "linear":
        n = x + w + y * (1 + bool(case.get("residual")) + bool(case.get("save")))
        return dict(bytes=n + (4 * N if case.get("bias") else 0), flops=2 * M * N * K)
    if op == "linear_backward":
        # dy, the pre-activation (where there is an activation), x and w in; dx, dw, dbias out
        n = y * (1 + (case.get("act", "none") != "none")) + 2 * x + 2 * w
        return dict(bytes=n + (4 * N if case.get("bias") else 0), flops=4 * M * N * K)
    if op == "gated":
        return dict(bytes=x + 2 * w + y * (3 if case.get("save") else 1), flops=4 * M * N * K)
    # dh, gate, up, x and both weights in; dx and both weights' gradients out
    return dict(bytes=3 * y + 2 * x + 4 * w, flops=8 * M * N * K)


# ---- inputs -------------------------------------------------------------------


def _empty(rows, cols, dtype):
    """rows x cols whose row pitch is cols rounded up to eight elements."""
    return torch.empty(rows, -(-cols // 8) * 8, dtype=dtype, device="cuda")[:, :cols]


class _Maker:
    def __init__(self, case, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(1_000_003 * seed + 17)
        self.dtype = DTYPES[case["dtype"]]

    def normal(self, rows, cols, std=1.0, dtype=None):
        t = _empty(rows, cols, dtype or self.dtype)
        t.copy_(torch.randn(rows, cols, generator=self.g, device="cuda").mul_(std))
        return t

    def weight(self, case):
        N, K = case["N"], case["K"]
        return self.normal(N, K, K ** -0.5) if case["rows"] else self.normal(K, N, K ** -0.5)


def prepare(case, seed):
    mk = _Maker(case, seed)
    M, N, K, dt = case["M"], case["N"], case["K"], mk.dtype
    s = dict(case=case, x=mk.normal(M, K))
    if case["op"].startswith("linear"):
        s["w"] = mk.weight(case)
        # Biases are kept in 32 bits.
        s["bias"] = mk.normal(1, N, 0.5, torch.float32)[0] if case["bias"] else None
        if case["op"] == "linear":
            s["residual"] = mk.normal(M, N) if case["residual"] else None
            s["y"] = _empty(M, N, dt)
            s["z"] = _empty(M, N, dt) if case["save"] else None
        else:
            # The upstream gradient, and the pre-activation the forward pass kept.
            s["dy"] = mk.normal(M, N)
            s["z"] = mk.normal(M, N, 1.1) if case["act"] != "none" else None
            s["dz"] = _empty(M, N, dt) if case["act"] != "none" else None
            s["dx"], s["dw"] = _empty(M, K, dt), torch.empty_strided(s["w"].shape, s["w"].stride(), dtype=dt,
                                                                     device="cuda")
            s["dbias"] = torch.empty(N, dtype=torch.float32, device="cuda") if case["bias"] else None
        return s
    s["wg"], s["wu"] = mk.weight(case), mk.weight(case)
    if case["op"] == "gated":
        s["h"] = _empty(M, N, dt)
        s["g"], s["u"] = (_empty(M, N, dt), _empty(M, N, dt)) if case["save"] else (None, None)
        return s
    s["dh"] = mk.normal(M, N)
    s["g"], s["u"] = mk.normal(M, N), mk.normal(M, N)
    s["dg"], s["du"] = _empty(M, N, dt), _empty(M, N, dt)
    s["dx"] = _empty(M, K, dt)
    s["dwg"], s["dwu"] = (torch.empty_strided(s[k].shape, s[k].stride(), dtype=dt, device="cuda")
                          for k in ("wg", "wu"))
    return s


# ---- the plain form -------------------------------------------------------------

_TANH_A, _TANH_B = math.sqrt(2.0 / math.pi), 0.044715


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return 0.5 * z * (1.0 + torch.tanh(_TANH_A * (z + _TANH_B * z * z * z)))


def _act_grad(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return 1.0 - (z <= 0).to(z.dtype)
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return sig * (1.0 + z * (1.0 - sig))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    t = torch.tanh(_TANH_A * (z + _TANH_B * z * z * z))
    return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * _TANH_A * (1.0 + 3.0 * _TANH_B * z * z)


def _plain(s):
    case = s["case"]
    dt, act, rows = s["x"].dtype, case["act"], case["rows"]
    x = s["x"].float()
    if case["op"] == "linear":
        w = s["w"].float()
        z = x @ (w.t() if rows else w)
        if s["bias"] is not None:
            z = z + s["bias"]
        y = _act(z, act)
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return (y.to(dt), z.to(dt)) if s["z"] is not None else y.to(dt)
    if case["op"] == "linear_backward":
        w, dz = s["w"].float(), s["dy"].float()
        if s["z"] is not None:
            dz = dz * _act_grad(s["z"].float(), act)
        dx = dz @ (w if rows else w.t())
        dw = dz.t() @ x if rows else x.t() @ dz
        out = [dx.to(dt), dw.to(dt)]
        if s["dbias"] is not None:
            out.append(dz.double().sum(0).float())
        return out
    wg, wu = s["wg"].float(), s["wu"].float()
    if case["op"] == "gated":
        g, u = x @ (wg.t() if rows else wg), x @ (wu.t() if rows else wu)
        h = _act(g, act) * u
        return (h.to(dt), g.to(dt), u.to(dt)) if s["g"] is not None else h.to(dt)
    g, u, dh = s["g"].float(), s["u"].float(), s["dh"].float()
    dg, du = dh * u * _act_grad(g, act), dh * _act(g, act)
    dx = dg @ (wg if rows else wg.t()) + du @ (wu if rows else wu.t())
    if rows:
        return dx.to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt)
    return dx.to(dt), (x.t() @ dg).to(dt), (x.t() @ du).to(dt)


# ---- through the framework --------------------------------------------------------

_kernels = None


def _own(s):
    global _kernels
    if _kernels is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "cuda-ir.go_b200"))
        from cudair import kernels
        _kernels = kernels
    k, case = _kernels, s["case"]
    act, rows = case["act"], case["rows"]
    if case["op"] == "linear":
        k.linear(s["x"], s["w"], s["y"], bias=s["bias"], residual=s["residual"], z=s["z"], act=act, b_trans=rows)
        return (s["y"], s["z"]) if s["z"] is not None else s["y"]
    if case["op"] == "linear_backward":
        k.linear_backward(s["dy"], s["x"], s["w"], z=s["z"], dz=s["dz"], da=s["dx"], db=s["dw"], dbias=s["dbias"],
                          act=act, b_trans=rows)
        return [s["dx"], s["dw"]] + ([s["dbias"]] if s["dbias"] is not None else [])
    if case["op"] == "gated":
        k.gated(s["x"], s["wg"], s["wu"], s["h"], g=s["g"], u=s["u"], act=act, b_trans=rows)
        return (s["h"], s["g"], s["u"]) if s["g"] is not None else s["h"]
    k.gated_backward(s["dh"], s["x"], s["wg"], s["wu"], s["g"], s["u"], s["dg"], s["du"], dx=s["dx"],
                     dwg=s["dwg"], dwu=s["dwu"], act=act, b_trans=rows)
    return s["dx"], s["dwg"], s["dwu"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- 64 bits ----------------------------------------------------------------------


def exact(case, seed):
    """The definition in 64 bits; gradients by differentiating the forward
    definition."""
    s = prepare(case, seed)
    fn = {"none": lambda t: t, "relu": torch.relu, "silu": torch.nn.functional.silu,
          "gelu": torch.nn.functional.gelu,
          "gelu_tanh": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[case["act"]]
    eq = "mk,nk->mn" if case["rows"] else "mk,kn->mn"
    x = s["x"].double()

    def pull(y, leaves, dy):
        return torch.autograd.grad(y, leaves, dy)

    if case["op"] == "linear":
        z = torch.einsum(eq, x, s["w"].double())
        z = z if s["bias"] is None else z + s["bias"].double()
        y = fn(z)
        y = y if s["residual"] is None else y + s["residual"].double()
        return (y, z) if s["z"] is not None else y
    if case["op"] == "linear_backward":
        dz = s["dy"].double()
        if s["z"] is not None:
            z = s["z"].double().requires_grad_()
            dz, = pull(fn(z), [z], dz)
        x, w = x.requires_grad_(), s["w"].double().requires_grad_()
        got = list(pull(torch.einsum(eq, x, w), [x, w], dz))
        return got + ([dz.sum(0)] if s["dbias"] is not None else [])
    if case["op"] == "gated":
        g, u = torch.einsum(eq, x, s["wg"].double()), torch.einsum(eq, x, s["wu"].double())
        h = fn(g) * u
        return (h, g, u) if s["g"] is not None else h
    g, u = s["g"].double().requires_grad_(), s["u"].double().requires_grad_()
    dg, du = pull(fn(g) * u, [g, u], s["dh"].double())
    x, wg, wu = x.requires_grad_(), s["wg"].double().requires_grad_(), s["wu"].double().requires_grad_()
    return pull([torch.einsum(eq, x, wg), torch.einsum(eq, x, wu)], [x, wg, wu], [dg, du])

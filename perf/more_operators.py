"""The measured workloads of the operators of a token block's second half.

Two operators: ``norm`` (layer norm, alone or of the sum with a residual
stream, with the reduction of its weight's and bias's gradients) and ``gated``
(the two projections of a gated feed-forward, the activation and the product).
``train`` cases run the forward and the gradients for given upstream gradients,
the others the forward alone.  Rows are tokens.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
EPS = 1e-5
ACTIVATIONS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


def listed():
    return [
        # One new token for each of eight sequences being answered, with the
        # stream that the block before adds to: all launch and latency.
        _norm(name="norm_token_bf16", rows=8, width=2048, dtype="bf16", residual=True, train=False),
        # The norm in front of a training step's feed-forward.
        _norm(name="norm_train_bf16", rows=16384, width=2048, dtype="bf16", residual=True,
              train=True),
        # Rows wider than a workgroup holds in few registers, without a stream.
        _norm(name="norm_wide_fp16", rows=3000, width=16384, dtype="fp16", residual=False,
              train=True),
        # Odd in both sizes, in single precision (a small model's training).
        _norm(name="norm_odd_fp32", rows=5013, width=1001, dtype="fp32", residual=False,
              train=True),
        # A prompt's tokens, forward only.
        _norm(name="norm_prompt_bf16", rows=4096, width=4096, dtype="bf16", residual=True,
              train=False),
        # One token: both matrices are read for a single row.
        _gated(name="gated_token_bf16", rows=1, width=2048, hidden=8192, dtype="bf16",
               activation="silu", train=False),
        # A step of many sequences that are answered together, of uneven sizes.
        _gated(name="gated_step_fp16", rows=45, width=4096, hidden=11000, dtype="fp16",
               activation="gelu_tanh", train=False),
        # A long prompt through a large block.
        _gated(name="gated_prompt_bf16", rows=8192, width=4096, hidden=16384, dtype="bf16",
               activation="silu", train=False),
        # Training steps of two sizes.
        _gated(name="gated_train_bf16", rows=8192, width=2048, hidden=8192, dtype="bf16",
               activation="silu", train=True),
        _gated(name="gated_train_fp16", rows=4096, width=1024, hidden=4096, dtype="fp16",
               activation="gelu", train=True),
        # Packed rows, no size a multiple of a tile or of a vector.
        _gated(name="gated_odd_bf16", rows=1025, width=1001, hidden=2731, dtype="bf16",
               activation="gelu", train=True),
        # Single precision.
        _gated(name="gated_train_fp32", rows=2048, width=1024, hidden=2816, dtype="fp32",
               activation="silu", train=True),
    ]


def _norm(name=None, *, rows, width, dtype, residual, train, affine=True):
    c = {"op": "norm", "rows": rows, "width": width, "dtype": dtype, "residual": residual,
         "train": train, "affine": affine}
    return {"name": name, **c} if name else c


def _gated(name=None, *, rows, width, hidden, dtype, activation, train):
    c = {"op": "gated", "rows": rows, "width": width, "hidden": hidden, "dtype": dtype,
         "activation": activation, "train": train}
    return {"name": name, **c} if name else c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    train = rng.random() < 0.6
    if rng.random() < 0.45:
        width = _log(rng, 16, 16384)
        if rng.random() < 0.5:
            width = max(1, width // 16) * 16
        rows = _log(rng, 1, max(1, min(65536, (1 << 25) // width)))
        return _norm(rows=rows, width=width, dtype=dtype, residual=rng.random() < 0.5, train=train,
                     affine=rng.random() < 0.8)
    width, hidden = _log(rng, 48, 4096), _log(rng, 96, 12000)
    if rng.random() < 0.6:
        width, hidden = max(1, width // 16) * 16, max(1, hidden // 16) * 16
    most = (1 << 37) // (width * hidden * (3 if train else 1))
    rows = _log(rng, 1, max(1, min(8192, most)))
    return _gated(rows=rows, width=width, hidden=hidden, dtype=dtype,
                  activation=rng.choice(ACTIVATIONS), train=train)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, by=1.0, plus=0.0):
        return (torch.randn(shape, generator=g, device=DEV) * by + plus).to(dt)

    state, M, K = {"case": case}, case["rows"], case["width"]
    if case["op"] == "norm":
        # a stream has a mean of its own, and some columns far larger than the rest
        scale = 1 + 15 * (torch.rand(K, generator=g, device=DEV) < 0.01)
        state["x"] = (torch.randn(M, K, generator=g, device=DEV) * scale + 0.3).to(dt)
        if case["residual"]:
            state["residual"] = (torch.randn(M, K, generator=g, device=DEV) * scale).to(dt)
        if case["affine"]:
            state["weight"], state["bias"] = normal(K, by=0.1, plus=1.0), normal(K, by=0.1)
        if case["train"]:
            state["gy"] = normal(M, K)
            if case["residual"]:
                state["gs"] = normal(M, K)
        return state
    F = case["hidden"]
    state["x"] = normal(M, K)
    state["gate"], state["up"] = normal(F, K, by=K ** -0.5), normal(F, K, by=K ** -0.5)
    if case["train"]:
        state["gh"] = normal(M, F, by=2.0 ** -6)  # as a loss's mean over tokens leaves them small
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _leaves(state, names, grad, dtype=None):
    """The state's tensors, cast, as new leaves of a graph where it trains."""
    out = {}
    for n in names:
        if n in state:
            t = state[n] if dtype is None else state[n].to(dtype)
            out[n] = t.detach().requires_grad_(grad)
    return out


def _finish(state, out, leaves, upstream):
    """Outputs, and in training the leaves' gradients, in the inputs' type."""
    dt = DTYPES[state["case"]["dtype"]]
    if not state["case"]["train"]:
        return {k: v.to(dt) for k, v in out.items()}
    grads = torch.autograd.grad([out[k] for k in out], list(leaves.values()),
                                [upstream[k].to(out[k].dtype) for k in out])
    return {**{k: v.detach().to(dt) for k, v in out.items()},
            **{"grad_" + k: g.to(dt) for k, g in zip(leaves, grads)}}


NORM_LEAVES = ("x", "residual", "weight", "bias")


class _Rounded(torch.autograd.Function):
    """The stream is kept in its type, and the norm is of what is kept."""

    @staticmethod
    def forward(ctx, s, dt):
        return s.to(dt).float()

    @staticmethod
    def backward(ctx, g):
        return g, None


def _plain_norm(state):
    case = state["case"]
    t = _leaves(state, NORM_LEAVES, case["train"], torch.float32)
    s = t["x"]
    if case["residual"]:
        s = _Rounded.apply(s + t["residual"], DTYPES[case["dtype"]])
    c = s - s.mean(-1, keepdim=True)
    y = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    if case["affine"]:
        y = y * t["weight"] + t["bias"]
    out, up = {"y": y}, {"y": state.get("gy")}
    if case["residual"]:
        out["s"], up["s"] = s, state.get("gs")
    return _finish(state, out, t, up)


def _activated(g, activation):
    if activation == "silu":
        return g / (1 + torch.exp(-g))
    if activation == "gelu":
        return 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    if activation == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    if activation == "relu":
        return g.clamp_min(0)
    return 1 / (1 + torch.exp(-g))


def _plain_gated(state):
    case = state["case"]
    t = _leaves(state, ("x", "gate", "up"), case["train"], torch.float32)
    g, u = t["x"] @ t["gate"].t(), t["x"] @ t["up"].t()
    return _finish(state, {"h": _activated(g, case["activation"]) * u}, t, {"h": state.get("gh")})


def _own_norm(state):
    from neural_shift_cuda import layer_norm
    case = state["case"]
    t = _leaves(state, NORM_LEAVES, case["train"])
    y = layer_norm(t["x"], t.get("weight"), t.get("bias"), residual=t.get("residual"), eps=EPS)
    if not case["residual"]:
        return _finish(state, {"y": y}, t, {"y": state.get("gy")})
    return _finish(state, {"y": y[0], "s": y[1]}, t, {"y": state.get("gy"), "s": state.get("gs")})


def _own_gated(state):
    from neural_shift_cuda import gated_linear
    case = state["case"]
    t = _leaves(state, ("x", "gate", "up"), case["train"])
    h = gated_linear(t["x"], t["gate"], t["up"], activation=case["activation"])
    return _finish(state, {"h": h}, t, {"h": state.get("gh")})


_PLAIN = {"norm": _plain_norm, "gated": _plain_gated}
_OWN = {"norm": _own_norm, "gated": _own_gated}


def run(state):
    case = state["case"]
    with torch.set_grad_enabled(case["train"]):
        return (_OWN if own else _PLAIN)[case["op"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    b, M, K = BYTES[case["dtype"]], case["rows"], case["width"]
    if case["op"] == "norm":
        # forward: the input (and the stream) read, the norm (and the sum) written;
        # gradients: the upstream ones read, one written (the input's and the
        # stream's are the same), the input read again as a forward came between
        n = (4 if case["residual"] else 2) + ((4 if case["residual"] else 3) if case["train"] else 0)
        return {"bytes": n * M * K * b + (4 if case["train"] else 2) * K * b * case["affine"],
                "flops": M * K * (20 if case["train"] else 8)}
    F = case["hidden"]
    once = (M * K + 2 * F * K + M * F) * b  # x, both matrices, h; then their gradients
    return {"bytes": once * (2 if case["train"] else 1), "flops": 4 * M * F * K * (3 if case["train"] else 1)}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_norm(state):
    case = state["case"]
    K = case["width"]
    s = state["x"].double()
    if case["residual"]:
        s = (s + state["residual"].double()).to(DTYPES[case["dtype"]]).double()
    var, mean = torch.var_mean(s, -1, correction=0, keepdim=True)
    hat = (s - mean) / torch.sqrt(var + EPS)
    w = state["weight"].double() if case["affine"] else torch.ones(K, dtype=torch.float64, device=DEV)
    out = {"y": torch.addcmul(state["bias"].double(), hat, w) if case["affine"] else hat}
    if case["residual"]:
        out["s"] = s
    if not case["train"]:
        return out
    gy = state["gy"].double()
    gw = gy * w
    along = (gw * hat).sum(-1, keepdim=True) / K
    grad = (gw - gw.sum(-1, keepdim=True) / K - hat * along) / torch.sqrt(var + EPS)
    if case["residual"]:
        grad = grad + state["gs"].double()
    out["grad_x"] = grad
    if case["residual"]:
        out["grad_residual"] = grad
    if case["affine"]:
        out["grad_weight"], out["grad_bias"] = (gy * hat).sum(0), gy.sum(0)
    return out


def _act(g, kind):
    """The activation and its slope."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if kind == "gelu":
        below = 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
        return g * below, below + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        a = 2 * math.sqrt(2 / math.pi)
        s = torch.sigmoid(a * (g + 0.044715 * g ** 3))
        return g * s, s + g * s * (1 - s) * a * (1 + 3 * 0.044715 * g * g)
    if kind == "relu":
        return torch.where(g > 0, g, 0.0), (g > 0).double()
    s = torch.sigmoid(g)
    return s, s * (1 - s)


def _exact_gated(state):
    """Some rows at a time."""
    case = state["case"]
    M, F, K = case["rows"], case["hidden"], case["width"]
    wg, wu = state["gate"].double(), state["up"].double()
    out = {"h": torch.empty(M, F, dtype=torch.float64, device=DEV)}
    if case["train"]:
        out["grad_x"] = torch.empty(M, K, dtype=torch.float64, device=DEV)
        out["grad_gate"], out["grad_up"] = torch.zeros_like(wg), torch.zeros_like(wu)
    for i in range(0, M, 2048):
        x = state["x"][i:i + 2048].double()
        g, u = torch.mm(x, wg.t()), torch.mm(x, wu.t())
        a, slope = _act(g, case["activation"])
        out["h"][i:i + 2048] = a * u
        if case["train"]:
            gh = state["gh"][i:i + 2048].double()
            dg, du = gh * u * slope, gh * a
            out["grad_x"][i:i + 2048] = torch.mm(dg, wg) + torch.mm(du, wu)
            out["grad_gate"] += torch.mm(dg.t(), x)
            out["grad_up"] += torch.mm(du.t(), x)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "gated": _exact_gated}[case["op"]](state)

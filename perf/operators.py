"""The measured workloads of the token operators.

Three operators: ``norm`` (per-head norm of queries and keys with the position
rotation), ``bias`` (a learned relative position bias by buckets, written out)
and ``attention`` (capped, biased and masked attention, for prompts, training
and single tokens over a cache).  ``train`` cases run the forward and the
gradients for given upstream gradients.  Tensors are (B, heads, tokens, width).
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}


def listed():
    return [
        # One new token for each of eight sequences being answered: the call
        # before the cache is written, all launch and latency.
        _norm(name="norm_token_bf16", B=8, Hq=32, Hk=8, L=1, D=128, rot=128, dtype="bf16",
              train=False),
        # A training step's queries and keys, as a projection leaves them
        # (tokens before heads, read through a transposed view).
        _norm(name="norm_train_bf16", B=4, Hq=16, Hk=4, L=4096, D=128, rot=128, dtype="bf16",
              train=True),
        # Odd everything in single precision: half of the width rotated, pairs
        # side by side.
        _norm(name="norm_odd_fp32", B=3, Hq=6, Hk=6, L=1025, D=80, rot=40, dtype="fp32",
              train=True, interleaved=True),
        # A bias shared by a model's layers, written out once a step.
        _bias(name="bias_train_fp32", H=16, Lq=2048, Lk=2048, buckets=32, reach=128, both=True,
              dtype="fp32", train=True),
        # The same for a short piece against a longer past, forward only.
        _bias(name="bias_rows_bf16", H=12, Lq=77, Lk=1001, buckets=64, reach=256, both=False,
              dtype="bf16", train=False),
        # Causal training with capped scores, four query heads to a key head.
        _attention(name="causal_cap_train_bf16", B=2, Hq=16, Hk=4, Lq=4096, Lk=4096, D=128,
                   dtype="bf16", train=True, causal=True, cap=50.0),
        # Documents packed into rows with padding at the end, linear distance
        # bias.
        _attention(name="packed_train_fp16", B=2, Hq=12, Hk=12, Lq=2500, Lk=2500, D=64,
                   dtype="fp16", train=True, causal=True, docs=7, slopes=True),
        # Patch tokens that all see each other, with the learned bias and its
        # gradient.
        _attention(name="buckets_train_bf16", B=4, Hq=12, Hk=12, Lq=1024, Lk=1024, D=64,
                   dtype="bf16", train=True, buckets=32, reach=128),
        # Single precision, odd lengths, queries the last third of the keys.
        _attention(name="odd_train_fp32", B=2, Hq=5, Hk=5, Lq=333, Lk=517, D=72, dtype="fp32",
                   train=True, cap=30.0, buckets=16, reach=64, degree=True),
        # A long prompt whose first part is seen from everywhere (an image
        # before its text).
        _attention(name="prefix_prompt_bf16", B=1, Hq=16, Hk=8, Lq=8192, Lk=8192, D=96,
                   dtype="bf16", train=False, causal=True, prefix=0.25),
        # One token against a long cache, sequences of different lengths.
        _attention(name="token_long_bf16", B=16, Hq=32, Hk=8, Lq=1, Lk=8192, D=128, dtype="bf16",
                   train=False, causal=True, cap=30.0, lengths=True),
        # One token against a short cache.
        _attention(name="token_short_fp16", B=1, Hq=8, Hk=8, Lq=1, Lk=500, D=64, dtype="fp16",
                   train=False, causal=True, slopes=True),
    ]


def _norm(name=None, *, B, Hq, Hk, L, D, rot, dtype, train, interleaved=False):
    c = {"op": "norm", "B": B, "Hq": Hq, "Hk": Hk, "L": L, "D": D, "rot": rot, "dtype": dtype,
         "train": train, "interleaved": interleaved}
    return {"name": name, **c} if name else c


def _bias(name=None, *, H, Lq, Lk, buckets, reach, both, dtype, train):
    c = {"op": "bias", "H": H, "Lq": Lq, "Lk": Lk, "buckets": buckets, "reach": reach,
         "both": both, "dtype": dtype, "train": train}
    return {"name": name, **c} if name else c


def _attention(name=None, *, B, Hq, Hk, Lq, Lk, D, dtype, train, causal=False, cap=0.0,
               prefix=0.0, docs=0, lengths=False, slopes=False, buckets=0, reach=0, degree=False):
    c = {"op": "attention", "B": B, "Hq": Hq, "Hk": Hk, "Lq": Lq, "Lk": Lk, "D": D,
         "dtype": dtype, "train": train, "causal": causal, "cap": cap, "prefix": prefix,
         "docs": docs, "lengths": lengths, "slopes": slopes, "buckets": buckets, "reach": reach,
         "degree": degree}
    return {"name": name, **c} if name else c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    D = rng.choice([16, 32, 40, 64, 72, 80, 96, 112, 128])
    Hk = _log(rng, 1, 12)
    Hq = Hk * rng.choice([1, 1, 2, 4])
    kind = rng.choice(["norm", "bias", "token", "prompt", "train", "train"])
    if kind == "norm":
        L = _log(rng, 1, 4096)
        B = _log(rng, 1, max(1, min(16, (1 << 18) // (L * Hq))))
        return _norm(B=B, Hq=Hq, Hk=Hk, L=L, D=D, rot=D if rng.random() < 0.6 else D // 4 * 2,
                     dtype=dtype, train=rng.random() < 0.6, interleaved=rng.random() < 0.3)
    if kind == "bias":
        Lq = _log(rng, 1, 2048)
        return _bias(H=Hq, Lq=Lq, Lk=_log(rng, Lq, max(2048, Lq)), buckets=rng.choice([16, 32, 64]),
                     reach=rng.choice([64, 128, 300, 1000]), both=rng.random() < 0.5, dtype=dtype,
                     train=rng.random() < 0.6)
    if kind == "token":
        Lk = _log(rng, 1, 8192)
        more = rng.random() < 0.5
        return _attention(B=_log(rng, 1, 16), Hq=Hq, Hk=Hk, Lq=1, Lk=Lk, D=D, dtype=dtype,
                          train=False, causal=True, cap=rng.choice([0.0, 30.0]), lengths=more,
                          slopes=rng.random() < 0.3, degree=rng.random() < 0.2)
    train = kind == "train"
    Lq = _log(rng, 1, 2048 if dtype != "fp32" else 700)
    Lk = Lq if rng.random() < 0.6 else _log(rng, Lq, 2 * Lq + 100)
    B = max(1, min(4, (1 << 26) // (Lq * Lk * Hq)))
    mask = rng.choice(["none", "causal", "causal", "prefix", "docs", "lengths"])
    bias = rng.choice(["none", "none", "slopes", "buckets"])
    return _attention(B=B, Hq=Hq, Hk=Hk, Lq=Lq, Lk=Lk, D=D, dtype=dtype, train=train,
                      causal=mask in ("causal", "prefix") or (mask == "docs" and rng.random() < 0.5),
                      cap=rng.choice([0.0, 30.0, 50.0]), prefix=0.3 if mask == "prefix" else 0.0,
                      docs=_log(rng, 2, 9) if mask == "docs" else 0, lengths=mask == "lengths",
                      slopes=bias == "slopes", buckets=32 if bias == "buckets" else 0,
                      reach=rng.choice([64, 128, 300]) if bias == "buckets" else 0,
                      degree=rng.random() < 0.3)


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _bucket_map(buckets, reach, both):
    """Bucket of each relative position -reach..reach: single steps near the
    query, then steps that grow with the logarithm of the distance; with
    ``both`` the second half of the buckets is for keys after the query,
    otherwise those share bucket 0."""
    n = buckets // 2 if both else buckets
    near = n // 2
    out = []
    for rel in range(-reach, reach + 1):
        d, first = (abs(rel), n if rel > 0 else 0) if both else (max(-rel, 0), 0)
        if d >= near:
            d = min(n - 1, near + int(math.log(d / near) / math.log(reach / near) * (n - near)))
        out.append(first + d)
    return out


def _lengths(case):
    """Filled part of each row's cache: from a half to the whole, in steps."""
    B, Lk = case["B"], case["Lk"]
    return [Lk - (Lk // 2) * i // max(1, B - 1) for i in range(B)] if case["lengths"] else [Lk] * B


def _documents(case):
    """Sizes of the documents packed into a row, and of the padding after them."""
    Lk, n = case["Lk"], case["docs"]
    pad = Lk // 50
    cuts = random.Random(n).choices(range(Lk - pad + 1), k=n - 1)
    cuts = [0] + sorted(cuts) + [Lk - pad]
    return [b - a for a, b in zip(cuts, cuts[1:])], pad


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV).to(dt)

    state = {"case": case}
    if case["op"] == "bias":
        state["table"] = normal(case["buckets"], case["H"])
        state["buckets"] = torch.tensor(_bucket_map(case["buckets"], case["reach"], case["both"]),
                                        dtype=torch.int32, device=DEV)
        if case["train"]:
            state["go"] = normal(case["H"], case["Lq"], case["Lk"])
        return state
    B, Hq, Hk, D = case["B"], case["Hq"], case["Hk"], case["D"]
    if case["op"] == "norm":
        L, rot = case["L"], case["rot"]
        # as a projection leaves them: tokens before heads
        state["q"] = normal(B, L, Hq, D).transpose(1, 2)
        state["k"] = normal(B, L, Hk, D).transpose(1, 2)
        state["wq"] = (1 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(dt)
        state["wk"] = (1 + 0.1 * torch.randn(D, generator=g, device=DEV)).to(dt)
        rows = 8192
        freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
        angle = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None] * freq
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        first = torch.randint(0, rows - L + 1, (B, 1), generator=g, device=DEV)
        state["positions"] = (first + torch.arange(L, device=DEV)).int()
        if case["train"]:
            state["gq"], state["gk"] = normal(B, Hq, L, D), normal(B, Hk, L, D)
        return state
    Lq, Lk = case["Lq"], case["Lk"]
    state["q"], state["k"], state["v"] = normal(B, Hq, Lq, D), normal(B, Hk, Lk, D), normal(B, Hk, Lk, D)
    rng = random.Random(seed)
    if case["lengths"]:
        n = _lengths(case)
        rng.shuffle(n)
        state["lengths"] = torch.tensor(n, dtype=torch.int32, device=DEV)
    if case["prefix"]:
        state["prefix"] = torch.full((B,), int(case["prefix"] * Lk), dtype=torch.int32, device=DEV)
    if case["docs"]:
        rows = []
        for _ in range(B):
            sizes, pad = _documents(case)
            rng.shuffle(sizes)
            rows.append(sum(([i] * s for i, s in enumerate(sizes)), []) + [-1] * pad)
        state["documents"] = torch.tensor(rows, dtype=torch.int32, device=DEV)
    if case["slopes"]:
        state["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)], device=DEV)
    if case["buckets"]:
        state["table"] = normal(case["buckets"], Hq)
        state["buckets"] = torch.tensor(_bucket_map(case["buckets"], case["reach"],
                                                    not case["causal"]),
                                        dtype=torch.int32, device=DEV)
    if case["train"]:
        state["go"] = normal(B, Hq, Lq, D)
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
    if not state["case"]["train"]:
        return out
    heads = [k for k in out if k in upstream]
    grads = torch.autograd.grad([out[k] for k in heads], list(leaves.values()),
                                [upstream[k].to(out[k].dtype) for k in heads])
    dt = DTYPES[state["case"]["dtype"]]
    return {**{k: v.detach() for k, v in out.items()},
            **{"grad_" + k: g.to(dt) for k, g in zip(leaves, grads)}}


def _rotate(x, cos, sin, interleaved):
    rot = 2 * cos.shape[-1]
    y, rest = x[..., :rot], x[..., rot:]
    a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:])
    c, s = cos[:, None], sin[:, None]
    a, b = a * c - b * s, a * s + b * c
    y = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((y, rest), -1)


def _plain_norm(state):
    case, dt = state["case"], DTYPES[state["case"]["dtype"]]
    t = _leaves(state, ("q", "k", "wq", "wk"), case["train"], torch.float32)
    cos, sin = state["cos"][state["positions"]], state["sin"][state["positions"]]
    out = {}
    for n in ("q", "k"):
        x = t[n]
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * t["w" + n]
        out[n] = _rotate(x, cos, sin, case["interleaved"])
    up = {"q": state.get("gq"), "k": state.get("gk")} if case["train"] else {}
    out = _finish(state, out, t, up)
    return {k: v.to(dt) for k, v in out.items()}


def _relative(Lq, Lk, lengths=None):
    """Relative position of key j to query i; the queries are the last of the
    keys (of each row's filled part)."""
    at = torch.arange(Lq, device=DEV)[:, None]
    j = torch.arange(Lk, device=DEV)[None]
    if lengths is None:
        return j - (at + Lk - Lq)
    return j - (at + (lengths.long()[:, None, None] - Lq))


def _plain_bias(state):
    case = state["case"]
    t = _leaves(state, ("table",), case["train"], torch.float32)
    rel = _relative(case["Lq"], case["Lk"]).clamp(-case["reach"], case["reach"]) + case["reach"]
    rows = state["buckets"].long()[rel]
    out = t["table"][rows].permute(2, 0, 1).contiguous()
    dt = DTYPES[case["dtype"]]
    if not case["train"]:
        return {"out": out.to(dt)}
    # the sum over the places of a bucket in 64 bits: it runs over millions
    n, up = case["buckets"], state["go"].double().flatten(1)
    grad = torch.zeros(case["H"], n, dtype=torch.float64, device=DEV)
    for b in range(n):
        grad[:, b] = (up * (rows.flatten() == b)).sum(1)
    return {"out": out.detach().to(dt), "grad_table": grad.t().to(dt)}


def _visible(state):
    case = state["case"]
    Lq, Lk = case["Lq"], case["Lk"]
    rel = _relative(Lq, Lk, state.get("lengths"))
    if rel.dim() == 2:
        rel = rel[None]
    j = torch.arange(Lk, device=DEV)
    ok = torch.ones_like(rel, dtype=torch.bool)
    if case["causal"]:
        ok = rel <= 0
    if "prefix" in state:
        ok = ok | (j < state["prefix"][:, None, None])
    if "lengths" in state:
        ok = ok & (j < state["lengths"][:, None, None])
    if "documents" in state:
        d = state["documents"]
        ok = ok & (d[:, Lk - Lq:, None] == d[:, None, :]) & (d[:, None, :] >= 0)
    return rel, ok  # (B or 1, Lq, Lk)


def _plain_attention(state):
    case, dt = state["case"], DTYPES[state["case"]["dtype"]]
    t = _leaves(state, ("q", "k", "v", "table"), case["train"], torch.float32)
    n = case["Hq"] // case["Hk"]
    k = t["k"].repeat_interleave(n, 1)
    v = t["v"].repeat_interleave(n, 1)
    s = torch.matmul(t["q"], k.transpose(2, 3).contiguous()) * case["D"] ** -0.5
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    rel, ok = _visible(state)
    if case["slopes"]:
        s = s - state["slopes"][:, None, None] * rel.abs()[:, None]
    if case["buckets"]:
        at = rel.clamp(-case["reach"], case["reach"]) + case["reach"]
        s = s + t["table"][state["buckets"].long()[at]].permute(0, 3, 1, 2)
    s = torch.where(ok[:, None], s, float("-inf"))
    m = s.detach().amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), 0.0, m)
    e = torch.exp(s - m)
    z = e.sum(-1, keepdim=True)
    out = {"out": torch.matmul(e / torch.where(z > 0, z, 1.0), v)}
    up = {"out": state["go"]} if case["train"] else {}
    if case["degree"]:
        out["degree"] = (m + torch.log(z)).squeeze(-1)
    degree = out.pop("degree").detach() if case["degree"] else None
    out = {k: x.to(dt) for k, x in _finish(state, out, t, up).items()}
    if degree is not None:
        out["degree"] = degree
    return out


def _own_norm(state):
    from neural_shift_cuda import qk_norm_rotary
    case = state["case"]
    t = _leaves(state, ("q", "k", "wq", "wk"), case["train"])
    q, k = qk_norm_rotary(t["q"], t["k"], t["wq"], t["wk"], state["cos"], state["sin"],
                          state["positions"], eps=1e-6, interleaved=case["interleaved"])
    up = {"q": state.get("gq"), "k": state.get("gk")} if case["train"] else {}
    return _finish(state, {"q": q, "k": k}, t, up)


def _own_bias(state):
    from neural_shift_cuda import relative_position_bias
    case = state["case"]
    t = _leaves(state, ("table",), case["train"])
    out = relative_position_bias(t["table"], state["buckets"], case["Lq"], case["Lk"])
    return _finish(state, {"out": out}, t, {"out": state.get("go")} if case["train"] else {})


def _own_attention(state):
    from neural_shift_cuda import biased_attention
    case = state["case"]
    t = _leaves(state, ("q", "k", "v", "table"), case["train"])
    out = biased_attention(t["q"], t["k"], t["v"], cap=case["cap"] or None,
                           causal=case["causal"], prefix=state.get("prefix"),
                           documents=state.get("documents"), lengths=state.get("lengths"),
                           slopes=state.get("slopes"), bias_table=t.get("table"),
                           buckets=state.get("buckets"), return_log_degree=case["degree"])
    out, degree = out if case["degree"] else (out, None)
    res = _finish(state, {"out": out}, t, {"out": state.get("go")} if case["train"] else {})
    return res if degree is None else {**res, "degree": degree.detach()}


_PLAIN = {"norm": _plain_norm, "bias": _plain_bias, "attention": _plain_attention}
_OWN = {"norm": _own_norm, "bias": _own_bias, "attention": _own_attention}


def run(state):
    case = state["case"]
    with torch.set_grad_enabled(case["train"]):
        return (_OWN if own else _PLAIN)[case["op"]](state)


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def _pairs(case):
    """Visible (query, key) pairs of one head, over the batch."""
    B, Lq, Lk = case["B"], case["Lq"], case["Lk"]
    if case["docs"]:
        sizes, _ = _documents(case)
        at, total, first = 0, 0, Lk - Lq  # queries of a document: those past `first`
        for s in sizes:
            q = max(0, at + s - max(at, first))
            total += q * s - (q * (q - 1) // 2 if case["causal"] else 0)
            at += s
        return B * total
    total, prefix = 0, int(case["prefix"] * Lk)
    for n in _lengths(case):
        if case["causal"]:
            total += sum(min(n, max(0, i + n - Lq + 1, min(prefix, n))) for i in range(Lq))
        else:
            total += Lq * n
    return total


def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "norm":
        n = case["B"] * case["L"] * (case["Hq"] + case["Hk"]) * case["D"]
        rows = case["B"] * case["L"] * case["rot"] * 4
        # forward: read, write; gradients: upstream read, gradients written
        # (q and k are read again only because a forward came between)
        return {"bytes": n * b * (4 if case["train"] else 2) + rows,
                "flops": n * (20 if case["train"] else 7)}
    if case["op"] == "bias":
        n = case["H"] * case["Lq"] * case["Lk"]
        return {"bytes": n * b * (2 if case["train"] else 1), "flops": n if case["train"] else 0}
    B, D = case["B"], case["D"]
    q = B * case["Hq"] * case["Lq"] * D * b
    kv = 2 * case["Hk"] * D * b * sum(_lengths(case))
    flops = 4 * D * case["Hq"] * _pairs(case)
    if not case["train"]:
        return {"bytes": 2 * q + kv, "flops": flops}
    return {"bytes": 4 * q + 2 * kv, "flops": 7 * flops // 2}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_norm(state):
    """Complex numbers turn, and the norm's gradient is written out."""
    case = state["case"]
    at = state["positions"].long()
    turn = torch.complex(state["cos"].double()[at], state["sin"].double()[at])[:, None]
    rot, il = case["rot"], case["interleaved"]

    def turned(x, by):
        y = x[..., :rot].unflatten(-1, (rot // 2, 2) if il else (2, rot // 2))
        z = torch.complex(y.select(-1 if il else -2, 0).contiguous(),
                          y.select(-1 if il else -2, 1).contiguous()) * by
        y = torch.stack((z.real, z.imag), -1 if il else -2).flatten(-2)
        return torch.cat((y, x[..., rot:]), -1)

    out = {}
    for n in ("q", "k"):
        x, w = state[n].double(), state["w" + n].double()
        r = (x.square().sum(-1, keepdim=True) / case["D"] + 1e-6) ** -0.5
        out[n] = turned(x * r * w, turn)
        if case["train"]:
            g = turned(state["g" + n].double(), turn.conj())  # a rotation's transpose
            out["grad_w" + n] = (g * x * r).sum((0, 1, 2))
            gw = g * w
            out["grad_" + n] = r * gw - x * r ** 3 * (gw * x).sum(-1, keepdim=True) / case["D"]
    order = ["q", "k"] + (["grad_q", "grad_k", "grad_wq", "grad_wk"] if case["train"] else [])
    return {k: out[k] for k in order}


def _exact_bias(state):
    """Diagonal by diagonal."""
    case = state["case"]
    Lq, Lk, R = case["Lq"], case["Lk"], case["reach"]
    table, ids = state["table"].double(), state["buckets"].tolist()
    ids = torch.tensor([ids[max(-R, min(R, d)) + R] for d in range(1 - Lk, Lk + 1)], device=DEV)
    line = table[ids]  # value of relative position d at d + Lk - 1
    first = [Lk - 1 - (i + Lk - Lq) for i in range(Lq)]
    out = torch.stack([line[f:f + Lk] for f in first]).permute(2, 0, 1).contiguous()
    if not case["train"]:
        return {"out": out}
    go, sums = state["go"].double(), torch.zeros_like(line)
    for i, f in enumerate(first):
        sums[f:f + Lk] += go[:, i].t()
    return {"out": out, "grad_table": torch.zeros_like(table).index_add_(0, ids, sums)}


def _exact_attention(state):
    """Head by head, with the gradients written out."""
    case = state["case"]
    B, Hq, D, cap = case["B"], case["Hq"], case["D"], case["cap"]
    per = Hq // case["Hk"]
    rel, ok = _visible(state)
    z = {n: torch.zeros(state[n].shape, dtype=torch.float64, device=DEV) for n in "qkv"}
    out = torch.zeros_like(z["q"])
    degree = torch.empty(out.shape[:3], dtype=torch.float64, device=DEV)
    if case["buckets"]:
        ids = state["buckets"].long()[rel[0].clamp(-case["reach"], case["reach"]) + case["reach"]] \
            if rel.shape[0] == 1 else None
        gt = torch.zeros(state["table"].shape, dtype=torch.float64, device=DEV)
    for b in range(B):
        see, d = ok[min(b, ok.shape[0] - 1)], rel[min(b, rel.shape[0] - 1)]
        for h in range(Hq):
            q, k, v = state["q"][b, h].double(), state["k"][b, h // per].double(), \
                state["v"][b, h // per].double()
            x = q @ k.t() / math.sqrt(D)
            y = cap * torch.tanh(x / cap) if cap else x
            s = y
            if case["slopes"]:
                s = s - state["slopes"][h].double() * d.abs()
            if case["buckets"]:
                row = ids if ids is not None else \
                    state["buckets"].long()[d.clamp(-case["reach"], case["reach"]) + case["reach"]]
                s = s + state["table"][:, h].double()[row]
            s = s.masked_fill(~see, -math.inf)
            degree[b, h] = torch.logsumexp(s, -1)
            p = torch.exp(s - degree[b, h][:, None]).masked_fill(~see, 0.0)
            out[b, h] = p @ v
            if not case["train"]:
                continue
            go = state["go"][b, h].double()
            z["v"][b, h // per] += p.t() @ go
            gs = p * (go @ v.t() - (go * out[b, h]).sum(-1, keepdim=True))
            if case["buckets"]:
                for n in range(gt.shape[0]):
                    gt[n, h] += (gs * (row == n)).sum()
            if cap:
                gs = gs * (1 - (y / cap) ** 2)
            gs = gs / math.sqrt(D)
            z["q"][b, h] = gs @ k
            z["k"][b, h // per] += gs.t() @ q
    res = {"out": out}
    if case["train"]:
        res.update(grad_q=z["q"], grad_k=z["k"], grad_v=z["v"])
        if case["buckets"]:
            res["grad_table"] = gt
    if case["degree"]:
        res["degree"] = degree
    return res


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "bias": _exact_bias,
                "attention": _exact_attention}[case["op"]](state)

"""biased_attention where its shared tiles run (a workgroup of 128 rows needs
one for every CU: many heads), and what reaches a row only through values that
are no numbers, the type's lowest bias, or offsets past 32 bits."""
from __future__ import annotations

import ctypes

import pytest
import torch

import token_oracle as oracle
from neural_shift_cuda import biased_attention, relative_buckets
from test_gpu_attention import DEV, TYPES, check, inputs, on_gpu

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
MANY = (4, 32, 32)  # x 2 row blocks: 256 workgroups


def rules_of(name, Lk, H, dtype, g):
    if name == "cap":
        return {"causal": True, "cap": 4.0}
    if name == "plain":
        return {}
    if name == "prefix":
        return {"causal": True, "cap": 300.0,
                "prefix": torch.tensor([0, 40, 100, 500], dtype=torch.int32)}
    if name == "lengths":
        return {"causal": True, "lengths": torch.tensor([Lk, 0, 77, 150], dtype=torch.int32)}
    if name == "documents":
        docs = (torch.arange(Lk) // 45).int().repeat(4, 1)
        docs[1, 160:] = -1
        docs[2] = torch.randint(-1, 3, (Lk,), generator=g)
        return {"documents": docs, "causal": True, "slopes": torch.rand(H, generator=g) / 4}
    buckets = relative_buckets(12, 30)
    return {"bias_table": torch.randn(12, H, generator=g).to(TYPES[dtype]), "buckets": buckets,
            "causal": name == "causal bias", "cap": 9.0 if name == "causal bias" else None}


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("name", ["plain", "cap", "prefix", "lengths", "documents", "bias",
                                  "causal bias"])
def test_shared_tiles(name, D, dtype):
    q, k, v, go, g = inputs(*MANY, 140, 200, D, dtype)
    check(q, k, v, go, rules_of(name, 200, 32, dtype, g))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_shared_tiles_with_shared_heads_and_degree(dtype):
    q, k, v, go, g = inputs(4, 32, 4, 200, 200, 72, dtype)
    check(q, k, v, go, {"causal": True, "scale": -0.3},
          gdegree=torch.randn(4, 32, 200, generator=g))


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("D", [32, 128])
def test_what_is_not_seen_adds_nothing(D, dtype, many):
    """No number in a key or an upstream row reaches what does not see it."""
    B, H, L, J = (4, 32, 140, 90) if many else (1, 2, 140, 90)
    q, k, v, go, _ = inputs(B, H, H, L, L, D, dtype)
    vals, tols = oracle.attention(q, k, v, go=go, causal=True)
    kb, vb = k.clone(), v.clone()
    kb[:, :, J], vb[:, :, J + 3] = float("nan"), float("inf")
    leaves = [t.to(DEV).requires_grad_() for t in (q, kb, vb)]
    out = biased_attention(*leaves, causal=True)
    gq = torch.autograd.grad(out, leaves[0], go.to(DEV))[0]
    oracle.close(out[:, :, :J], vals["out"][:, :, :J], tols["out"][:, :, :J], "out")
    oracle.close(gq[:, :, :J], vals["gq"][:, :, :J], tols["gq"][:, :, :J], "gq")
    assert out[:, :, J:].isnan().all()
    # an upstream gradient that is none: keys after its row do not see it
    bad = go.clone()
    bad[:, :, J] = float("inf")
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    gk, gv = torch.autograd.grad(biased_attention(*leaves, causal=True), leaves[1:], bad.to(DEV))
    for n, got in (("gk", gk), ("gv", gv)):
        oracle.close(got[:, :, J + 1:], vals[n][:, :, J + 1:], tols[n][:, :, J + 1:], n)


def test_rows_of_the_lowest_bias():
    """A row all of whose biases are the type's lowest value weighs its keys
    evenly, and its gradients are those of even weights."""
    q, k, v, go, _ = inputs(1, 2, 2, 70, 90, 32, "fp32")
    low = torch.full((1, 2), torch.finfo(torch.float32).min, device=DEV)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out = biased_attention(*leaves, bias_table=low, buckets=torch.zeros(1, dtype=torch.int32, device=DEV))
    gq, gk, gv = torch.autograd.grad(out, leaves, go.to(DEV))
    p = torch.full((1, 2, 70, 90), 1 / 90, dtype=torch.float64)
    Q, K, V, G = (t.double() for t in (q, k, v, go))
    dP = G @ V.transpose(2, 3)
    dX = p * (dP - (p * dP).sum(-1, keepdim=True)) * 32 ** -0.5
    # 200 roundings of the sums' magnitudes
    for got, want, size in ((out, p @ V, p @ V.abs()), (gq, dX @ K, dX.abs() @ K.abs()),
                            (gk, dX.transpose(2, 3) @ Q, dX.abs().transpose(2, 3) @ Q.abs()),
                            (gv, p.transpose(2, 3) @ G, p.transpose(2, 3) @ G.abs())):
        oracle.close(got, want, 200 * oracle.F32 * size + 1e-7, "even")


@pytest.mark.parametrize("lengths", [None, [0, 70]])
def test_gradients_from_the_degree_alone(lengths):
    """The native backward with log_degree in row_stats' place."""
    from neural_shift_cuda_amd import _C
    from neural_shift_cuda_amd.attention import _check_attention
    q, k, v, go, _ = inputs(2, 2, 2, 90, 90, 64, "bf16")
    rules = {"causal": True, "cap": 8.0}
    if lengths is not None:
        rules["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    vals, tols = oracle.attention(q, k, v, go=go, **rules)
    q, k, v, go = (t.to(DEV) for t in (q, k, v, go))
    r = on_gpu(rules)
    full = _check_attention(q, k, v, None, r["cap"], True, None, None, r.get("lengths"), None,
                            None, None)
    out, degree, _ = _C.attention_forward(q, k, v, full, True, False)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    a = _C._attention_args(q, k, v, out, degree, None, full)
    a.grad_out, a.go_stride = go.data_ptr(), go.stride()[:3]
    a.grad_q, a.grad_k, a.grad_v = (t.data_ptr() for t in grads)
    a.gq_stride, a.gk_stride, a.gv_stride = (t.stride()[:3] for t in grads)
    n = int(_C._lib.nsh_attention_workspace_bytes(ctypes.byref(a), 1))
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    a.workspace, a.workspace_bytes = ws.data_ptr(), n
    _C._call_on(q, "nsh_attention_backward", ctypes.byref(a))
    for name, g in zip(("gq", "gk", "gv"), grads):
        oracle.close(g, vals[name], tols[name], name)


def test_cache_past_32_bits():
    """One token over a cache of 2^31 elements a head: the last keys decide."""
    L, D, near = (1 << 24) + 700, 128, 512
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    k = torch.zeros(1, 1, L, D, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    g = torch.Generator().manual_seed(0)
    q, ke, ve = (torch.randn(1, 1, n, D, generator=g).bfloat16() for n in (1, near, near))
    k[:, :, -near:], v[:, :, -near:] = ke.to(DEV), ve.to(DEV)
    slopes = torch.tensor([2.0])  # e^-1000 and less beyond the last 512 keys
    out = biased_attention(q.to(DEV), k, v, causal=True, slopes=slopes.to(DEV))
    vals, tols = oracle.attention(q, ke, ve, causal=True, slopes=slopes)
    oracle.close(out, vals["out"], tols["out"], "out")


def test_far_token_strides_are_copied():
    q, k, v, go, _ = inputs(1, 1, 1, 5, 5, 32, "fp32")

    def far(t):
        room = torch.zeros(5, (1 << 22) + 64, device=DEV)
        room[:, :32] = t[0, 0].to(DEV)
        return room.as_strided((1, 1, 5, 32), (5 * room.shape[1], 5 * room.shape[1], room.shape[1], 1)).detach()

    check(q, k, v, go, {"causal": True}, layout=far)


def test_token_block():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "token_block.py")
    spec = importlib.util.spec_from_file_location("token_block", path)
    block = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(block)
    # the logits' sums of 128 products of unit size and the few steps behind them
    assert block.main(["--steps", "11"]) < 1e-4

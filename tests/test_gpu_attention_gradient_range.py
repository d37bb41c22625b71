"""Gradients in 16 bits at every size of the upstream ones: as near as the
type's own roundings, with nothing lost below its smallest normal number on the
way.

A rounding is off by at most u = eps / 2 of the value (u / sqrt(3) in the root
mean square at a binade's lower end), or by half of the type's smallest step;
dv has its weights' rounding and its own, dq and dk their own and in bf16 dx's.
A tenth more is for the spread over some thousand values, and 3.5 / sqrt(2 n)
over the n of one row."""
from __future__ import annotations

import math

import pytest
import torch

import token_dense as dense
import token_oracle as oracle
from neural_shift_cuda import biased_attention, relative_buckets
from test_gpu_attention import DEV, TYPES, inputs, on_gpu

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


def gradients(q, k, v, go, rules):
    """{name: (values, in 64 bits)}"""
    r, go = on_gpu(rules), go.to(DEV)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    vals = dense.attention(*leaves, go, **r)
    grads = torch.autograd.grad(biased_attention(*leaves, **r), leaves, go)
    return {n: (g.double(), vals[n]) for n, g in zip(("gq", "gk", "gv"), grads)}


def roundings(name, dtype):
    return 2 if name == "gv" or dtype is torch.bfloat16 else 1


def bound(want, n, dtype):
    """The root of the summed squares of n roundings of each of `want`."""
    u = torch.finfo(dtype).eps / 2
    return math.sqrt(n) * u / math.sqrt(3) * want.norm() + oracle.tiny(dtype) * math.sqrt(want.numel())


KINDS = {
    "plain": {},
    "causal": {"causal": True},
    "cap": {"cap": 20.0, "causal": True},
    "documents": {"documents": (torch.arange(900) // 350).int()[None]},
    "bias": {},
}


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,by", [("fp16", 0), ("fp16", -10), ("fp16", -14), ("fp16", -18),
                                      ("bf16", -14)])
def test_small_upstream_gradients(kind, D, dtype, by):
    rules = dict(KINDS[kind])
    q, k, v, go, g = inputs(1, 2, 2, 900, 900, D, dtype)
    if kind == "bias":
        rules.update(bias_table=torch.randn(32, 2, generator=g).to(TYPES[dtype]),
                     buckets=relative_buckets(32, 128))
    for name, (got, want) in gradients(q, k, v, go * 2.0 ** by, rules).items():
        err, most = (got - want).norm(), 1.1 * bound(want, roundings(name, TYPES[dtype]), TYPES[dtype])
        print(name, float(err / want.norm()), float(most / want.norm()))
        assert err <= most, (name, float(err / most))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L", [40, 700])  # rows in workgroups of 32 and 128; parts by keys
def test_rows_of_all_sizes(D, L):
    """Rows whose upstream gradients differ by up to 2^20: each row of dq has its own
    precision.  Documents of one row's size each have it for dk and dv too."""
    q, k, v, go, _ = inputs(1, 40, 40, L, L, D, "fp16")
    i = torch.arange(L)
    own = torch.float16
    got, want = gradients(q, k, v, (go * 2.0 ** -(i % 21).float()[:, None]).half(), {})["gq"]
    spread = 1.1 + 3.5 / math.sqrt(2 * D)
    for n in range(0, 21, 4):
        a, b = got[0, :, n::21], want[0, :, n::21]
        most = oracle.half_ulp(own) / math.sqrt(3) * b.norm(dim=-1) + oracle.tiny(own) * math.sqrt(D)
        assert ((a - b).norm(dim=-1) <= spread * most).all(), n
    docs = (i * 3 // L).int()[None]
    small = (go * 2.0 ** -(9.0 * docs[0])[:, None]).half()
    for name, (got, want) in gradients(q, k, v, small, {"documents": docs}).items():
        for d in range(3):
            a, b = (t[:, :, (docs[0] == d).to(DEV)] for t in (got, want))
            assert (a - b).norm() <= 1.1 * bound(b, roundings(name, own), own), (name, d)


@pytest.mark.parametrize("cap", [None, 40.0])
@pytest.mark.parametrize("D", [64, 128])
def test_large_upstream_gradients(cap, D):
    """dx beyond the type's largest number, where dq and dk are within it."""
    q, k, v, go, _ = inputs(1, 2, 2, 64, 64, D, "fp16")
    rules = {"scale": 1 / (2 * D), "cap": cap}
    for name, (got, want) in gradients(q * 4, k * 4, v * 64, go * 1024, rules).items():
        assert want.abs().max() < 60000
        assert (got - want).norm() <= 1.1 * bound(want, roundings(name, torch.float16), torch.float16), name


def test_weights_of_very_long_rows():
    """dv where every weight, 1 / 60000, is below fp16's smallest normal number."""
    n, D = 60000, 64
    g = torch.Generator().manual_seed(2)
    go = torch.randn(1, 1, 32, D, generator=g).half().abs()
    q, k = torch.zeros(1, 1, 32, D).half(), torch.zeros(1, 1, n, D).half()
    v = torch.randn(1, 1, n, D, generator=g).half()
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    # upstream gradients of 2^10, so that the results are normal numbers
    gv = torch.autograd.grad(biased_attention(*leaves), leaves, (go * 1024).to(DEV))[2]
    want = (go * 1024).double().sum(2, keepdim=True) / n
    u = torch.finfo(torch.float16).eps / 2
    assert ((gv.double().cpu() - want).abs() <= (2 * u + 2.0 ** -16) * want).all()

"""The gradients of biased_attention as wholes: no error that a row's pairs
share adds up past the roundings that the type itself brings.

A rounding is off by at most u = eps / 2 of the value, u / sqrt(3) in the root
mean square where every value is at its binade's lower end; n independent ones
give sqrt(n) times that.  The table's gradient is rounded once, at its end.  dv
has the weights' rounding and its own, dq and dk have dx's and their own (fp16
takes dx in two parts, which leaves their own).  A tenth more is for the spread
of a mean over some hundred values (the mean square of uniform errors is off by
0.9 / sqrt(count))."""
from __future__ import annotations

import math

import pytest
import torch

import token_oracle as oracle
from neural_shift_cuda import biased_attention, relative_buckets
from test_gpu_attention import DEV, TYPES, inputs, on_gpu

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("B,H,L,D", [(1, 16, 900, 64),     # rows in workgroups of 32
                                     (8, 16, 300, 128)])   # of 128
def test_no_shared_error(B, H, L, D, dtype):
    q, k, v, go, g = inputs(B, H, H, L, L, D, dtype)
    rules = {"bias_table": torch.randn(32, H, generator=g).to(TYPES[dtype]),
             "buckets": relative_buckets(32, 128)}
    vals, _ = oracle.attention(q, k, v, go=go, **rules)
    r = on_gpu(rules)
    table = r["bias_table"].requires_grad_()
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)] + [table]
    out = biased_attention(*leaves[:3], bias_table=table, buckets=r["buckets"])
    grads = torch.autograd.grad(out, leaves, go.to(DEV))
    u = torch.finfo(TYPES[dtype]).eps / 2
    pair = 2 if dtype == "bf16" else 1
    for name, got, n in zip(("gq", "gk", "gv", "gtable"), grads, (pair, pair, 2, 1)):
        want = vals[name].double().cpu()
        err = ((got.double().cpu() - want).norm() / want.norm()).item()
        print(name, err)
        assert err <= 1.1 * math.sqrt(n) * u / math.sqrt(3), (name, err)

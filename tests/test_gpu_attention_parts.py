"""Gradients by keys where a key block's queries are shared by more workgroups
than it has tiles of them: single heads, causal, whose last keys are seen by few
rows."""
from __future__ import annotations

import math

import pytest
import torch

import token_dense as dense
from neural_shift_cuda import biased_attention
from test_gpu_attention import DEV, inputs

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


def check(q, k, v, go, rules):
    """As wholes: the weights' or dx's rounding and the result's own, and a tenth."""
    rules = {n: t.to(DEV) if isinstance(t, torch.Tensor) else t for n, t in rules.items()}
    leaves, go = [t.to(DEV).requires_grad_() for t in (q, k, v)], go.to(DEV)
    want = dense.attention(*leaves, go, **rules)
    got = torch.autograd.grad(biased_attention(*leaves, **rules), leaves, go)
    u = torch.finfo(q.dtype).eps / 2
    for n, g in zip(("gq", "gk", "gv"), got):
        assert (g.double() - want[n]).norm() <= 1.1 * math.sqrt(2 / 3) * u * want[n].norm(), n
        # the last keys, whose rows are few
        a, b = g.double()[:, :, -128:], want[n][:, :, -128:]
        assert (a - b).norm() <= 1.2 * math.sqrt(2 / 3) * u * b.norm(), n


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [96, 128])
@pytest.mark.parametrize("cap", [None, 20.0])
def test_parts_without_rows(dtype, D, cap):
    q, k, v, go, _ = inputs(1, 1, 1, 1024, 1024, D, dtype)
    check(q, k, v, go, {"causal": True, "cap": cap})


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_parts_without_rows_of_a_short_cache(dtype):
    q, k, v, go, _ = inputs(2, 2, 1, 700, 900, 128, dtype)
    check(q, k, v, go, {"causal": True, "lengths": torch.tensor([900, 130], dtype=torch.int32)})

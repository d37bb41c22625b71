"""Gradients of calls without a bias whose scores are large: a row's weights add
up to one behind any maximum.

All keys of a row's half are one vector, so a row has n scores of one value and
n that lie `top` below it: its weights are 1 / n and e^-top / n.  Then dv = (the
sum of dO) / n for every key of the upper half and e^-top of that for the others."""
from __future__ import annotations

import math

import pytest
import torch

from neural_shift_cuda import biased_attention
from test_gpu_attention import DEV, TYPES

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("top", [50.0, 3e3, 1e5, 1.5e7])
@pytest.mark.parametrize("negative", [False, True])
def test_weights_add_up_to_one(dtype, D, top, negative):
    dt, Lq, n = TYPES[dtype], 70, 301  # 1 / n is no power of two
    g = torch.Generator().manual_seed(1)
    q = torch.ones(1, 2, Lq, D, dtype=dt)
    k = torch.cat((torch.ones(1, 2, n, D), torch.zeros(1, 2, n, D)), 2).to(dt)
    v = torch.randn(1, 2, 2 * n, D, generator=g).to(dt)
    go = torch.randn(1, 2, Lq, D, generator=g).to(dt)
    scale = top / D
    if negative:
        q, scale = -q, -scale
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out = biased_attention(*leaves, scale=scale)
    gv = torch.autograd.grad(out, leaves, go.to(DEV))[2].double().cpu()
    sums, size = go.double().sum(2, keepdim=True), go.double().abs().sum(2, keepdim=True)
    # the weight's and the result's roundings; an exponent's next to 1024 (16 bits)
    # and the sums' in fp32
    u = torch.finfo(dt).eps / 2
    loose = 64 * 2.0 ** -24 + (2.0 ** -14 if dt is not torch.float32 else 0.0)
    tol = (2 * u + loose) * size / n + torch.finfo(dt).smallest_normal
    assert ((gv[:, :, :n] - sums / n).abs() <= tol).all()
    low = gv[:, :, n:] - math.exp(-top) * sums / n
    assert (low.abs() <= tol * math.exp(-50.0) + torch.finfo(dt).smallest_normal).all()
    want = v.double()[:, :, :n].mean(2, keepdim=True)
    err = (out.double().cpu() - want).abs()
    assert (err <= (2 * u + loose) * v.double()[:, :, :n].abs().mean(2, keepdim=True)).all()

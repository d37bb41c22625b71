"""16-bit rows whose value lies in very many small weights next to one large one."""
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


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("Lq", [1, 200])          # shared keys, and workgroups of 128 rows
@pytest.mark.parametrize("where", [0, 70_000])    # the large one first, or behind half of the others
def test_many_small_weights(dtype, Lq, where):
    dt, n, D, heads = TYPES[dtype], 140_000, 64, 1 if Lq == 1 else 128
    top = 14.5  # the small weights, e^-top, are 8.46 of fp16's smallest steps
    k = torch.zeros(1, 1, n, D, device=DEV, dtype=dt)
    k[:, :, where] = 1
    v = torch.ones(1, 1, n, D, device=DEV, dtype=dt) * torch.linspace(0.5, 2.0, D, device=DEV).to(dt)
    v[:, :, where] = 0
    q = torch.ones(1, heads, Lq, D, device=DEV, dtype=dt)
    out, degree = biased_attention(q, k, v, scale=top / D, return_log_degree=True)
    share = (n - 1) / (n - 1 + math.exp(top))
    want = share * v[0, 0, where - 1].double()
    # the weights' and the result's roundings and the sums' in fp32: those of n / 64
    # tiles, one after the other
    u = torch.finfo(dt).eps / 2
    tol = (2 * u + (n / 64 + 64) * 2.0 ** -24) * want
    assert ((out.double() - want).abs() <= tol).all()
    assert (degree.double() - math.log(n - 1 + math.exp(top))).abs().max() <= (n / 64 + 64) * 2.0 ** -24

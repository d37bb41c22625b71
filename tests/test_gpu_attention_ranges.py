"""biased_attention at the ends of the caps it serves: a cap far above every
score is none, one far below leaves every key the same weight."""
from __future__ import annotations

import pytest
import torch

import token_dense as dense
from neural_shift_cuda import biased_attention
from test_gpu_attention import DEV, TYPES, inputs

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("Lq", [1, 40, 300])
@pytest.mark.parametrize("high", [True, False])
def test_ends_of_the_caps(dtype, Lq, high):
    q, k, v, go = (t.to(DEV) for t in inputs(1, 8, 8, Lq, 300, 64, dtype)[:4])
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = biased_attention(*leaves, causal=True, cap=2.0 ** (60 if high else -60))
    got = [out, *torch.autograd.grad(out, leaves, go)]
    want = dense.attention(q, k, v, go, causal=True, **({} if high else {"scale": 0.0}))
    u = torch.finfo(TYPES[dtype]).eps / 2
    for n, g in zip(("out", "gq", "gk", "gv") if high else ("out",), got):
        # the weights' or dx's rounding, the result's and the sums'
        assert (g.double() - want[n]).norm() <= (2 * u + 2.0 ** -18) * want[n].norm(), n
    assert all(g.isfinite().all() for g in got)


def test_beyond_them():
    q, k, v = (t.to(DEV) for t in inputs(1, 2, 2, 5, 9, 8, "fp32")[:3])
    for rules in ({"cap": 1e39}, {"cap": 1e-46}, {"scale": 1e39}):
        with pytest.raises(RuntimeError, match="within fp32"):
            biased_attention(q, k, v, **rules)

"""The gated projections in fp32 as sums of bf16 parts: what becomes of numbers beyond fp32."""
from __future__ import annotations

import pytest
import torch

from neural_shift_cuda import gated_linear

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda"
M, K, F = 2000, 132, 1100  # sizes that are taken apart (test_gpu_gated_parts.py)
INF = float("inf")


def full(*shape, seed):
    """Numbers of 24 bits in [1, 2)."""
    return 1.0 + torch.rand(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).float()


def run(x, gate, up, gh):
    leaves = [t.to(DEV).requires_grad_() for t in (x, gate, up)]
    h = gated_linear(*leaves, activation="relu")
    return dict(zip(("h", "gx", "ggate", "gup"), (h.detach(), *torch.autograd.grad(h, leaves, gh.to(DEV)))))


@pytest.mark.parametrize("size", [1e12, 1e25, 3e38])
def test_products_beyond_fp32(size):
    """Of one sign and far beyond fp32: an infinity of that sign, as in fp32."""
    rand = [full(*s, seed=i) for i, s in enumerate(((M, K), (F, K), (F, K), (M, F)))]
    x, gate, up, gh = rand
    x, up = x * 1e30, up * 1e-30
    assert not run(x, gate * (-size / 2), up, gh)["h"].any()
    assert (run(x, gate * (size / 2), up, gh)["h"] == INF).all()
    # gradients: g = u = 1, dg = du = gh
    x, one = torch.zeros(M, K), torch.zeros(F, K)
    x[:, 0] = one[:, 0] = 1.0
    big = rand[1] * (-size / 2)
    big[:, 0] = 1.0
    assert (run(x, big, big, gh * 1e30)["gx"][:, 1:] == -INF).all()
    x = rand[0] * (-size / 2)
    x[:, 0] = 1.0
    got = run(x, one, one, gh * 1e30)
    assert (got["ggate"][:, 1:] == -INF).all() and (got["gup"][:, 1:] == -INF).all()


def test_infinity_times_infinity():
    x, gate, up = full(M, K, seed=1), full(F, K, seed=2), full(F, K, seed=3)
    x[0, 0], x[7, 3], gate[5, 0], up[6, 3] = INF, -INF, INF, -INF
    want = (x.double() @ gate.double().t()).relu() * (x.double() @ up.double().t())
    got = run(x, gate, up, torch.zeros(M, F))["h"].cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]) and got[~inf & ~want.isnan()].isfinite().all()

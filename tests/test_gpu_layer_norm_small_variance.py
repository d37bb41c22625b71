"""layer_norm where the variance and eps together are below fp32's smallest normal number."""
from __future__ import annotations

import pytest
import torch

import block_oracle as oracle
from neural_shift_cuda import layer_norm

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [64, 600, 4096, 20000])
def test_small_deviations(n, dtype):
    """+-2^-66: squares of 2^-132, whose sum is exact, and the norm +-1 but for a root and a
    product."""
    x = torch.full((3, n), 2.0 ** -66, device=DEV, dtype=dtype)
    x[:, ::2] *= -1
    x.requires_grad_()
    y = layer_norm(x, eps=0.0)
    want = x.detach().sign().double().cpu()
    oracle.close(y, want, 4 * oracle.F32 + oracle.half_ulp(dtype) * want.abs(), "y")
    # gy = y: its gradient is that of a row's length, which the norm does not change
    (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert gx.isfinite().all()


def test_a_small_eps():
    """A row of one value is the bias for every eps above 0."""
    b = torch.randn(64, generator=torch.Generator().manual_seed(0)).to(DEV)
    x = torch.full((2, 64), 3.0, device=DEV)
    assert torch.equal(layer_norm(x, None, b, eps=2.0 ** -140), b.expand(2, 64))

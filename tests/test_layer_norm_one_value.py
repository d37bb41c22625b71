"""layer_norm of rows of one value: the norm is 0 and what comes out is the bias, however
large the value and however its sums round."""
from __future__ import annotations

import pytest
import torch

import block_oracle as oracle
from neural_shift_cuda import layer_norm

ON = ["cpu", pytest.param("cuda", marks=[
    pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")])]

# A mean is off by at most its longest chain of additions, 64 + n / 128 of them, in steps of the
# value's last place.  So are the deviations, and the sum of n of them has less than 2^24 of those
# steps: it is exact in whatever order, their mean is the deviation itself and what is left is 0.
VALUES = [(-1e9, 1e-5), (1.498e9, 1e-5), (60574.5, 1e-12)]
WIDTHS = [9, 100, 771, 1025, 1500, 2047, 3411, 3856, 4100, 6080, 8191, 8200, 20000]


def inputs(value, n, dtype=torch.float32):
    g = torch.Generator().manual_seed(n)
    w, b, gy = (torch.randn(*s, generator=g) for s in ((n,), (n,), (3, n)))
    return torch.full((3, n), value).to(dtype), w.to(dtype), b.to(dtype), gy.to(dtype)


@pytest.mark.parametrize("on", ON)
@pytest.mark.parametrize("value,eps", VALUES)
def test_the_bias_is_left(value, eps, on):
    for n in WIDTHS:
        for dtype in (torch.float32, torch.bfloat16):
            x, w, b, _ = (t.to(on) for t in inputs(value, n, dtype))
            assert torch.equal(layer_norm(x, w, b, eps=eps), b.expand(3, n)), (n, dtype)


@pytest.mark.parametrize("on", ON)
@pytest.mark.parametrize("value,eps", VALUES)
def test_gradients(value, eps, on):
    """gx = (t - mean(t)) / sqrt(eps), t = gy w; the squares of a narrow row's deviations have
    less than 2^24 steps too (42 of them squared, 1500 times), and the variance is 0."""
    for n in (9, 100, 771, 1500):
        x, w, b, gy = inputs(value, n)
        leaves = [t.to(on).requires_grad_() for t in (x, w, b)]
        gx, gw, gb = torch.autograd.grad(layer_norm(*leaves, eps=eps), leaves, gy.to(on))
        t = gy.double() * w.double()
        r = eps ** -0.5
        want = r * (t - t.mean(-1, keepdim=True))
        size = t.abs() + t.abs().mean(-1, keepdim=True)
        oracle.close(gx, want, r * (64 + n / 128 + 16) * oracle.F32 * size, f"gx {n}")
        assert not gw.any()
        oracle.close(gb, gy.double().sum(0), 4 * oracle.F32 * gy.double().abs().sum(0), f"gb {n}")

"""gated_linear where a formula's own value is infinite, 0 or empty."""
from __future__ import annotations

import pytest
import torch

from neural_shift_cuda import gated_linear

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda"
INF = float("inf")


def test_weights_of_no_width_in_any_order():
    for empty in (lambda n: torch.empty(n, 0, device=DEV), lambda n: torch.empty(0, n, device=DEV).t()):
        x, gate, up = (empty(n).requires_grad_() for n in (3, 5, 5))
        h = gated_linear(x, gate, up)
        assert h.shape == (3, 5) and not h.any()
        for g, t in zip(torch.autograd.grad(h.sum(), (x, gate, up)), (x, gate, up)):
            assert g.shape == t.shape


@pytest.mark.parametrize("dtype,M,F", [(torch.bfloat16, 70, 33), (torch.float16, 70, 33), (torch.float32, 70, 33),
                                       (torch.bfloat16, 2000, 1100), (torch.float32, 2000, 1100)])
def test_an_infinite_row_beside_a_ragged_end(dtype, M, F):
    """Positive numbers all over: an infinity in x makes its row of h and dx infinite, and its
    terms of the weights' gradients; the places past the last hidden column add nothing."""
    K = 132
    g = torch.Generator().manual_seed(F)
    x, gate, up, gh = ((torch.rand(*s, generator=g) + 0.5).to(dtype) for s in ((M, K), (F, K), (F, K), (M, F)))
    gate, up = gate / 128, up / 128
    x[3, 7] = INF
    leaves = [t.to(DEV).requires_grad_() for t in (x, gate, up)]
    h = gated_linear(*leaves, activation="relu")
    gx, gg, gu = torch.autograd.grad(h, leaves, gh.to(DEV))
    assert (h[3] == INF).all() and (gx[3] == INF).all()
    assert (gg == INF).all() and (gu == INF).all()
    rest = [m for m in range(M) if m != 3]
    assert h[rest].isfinite().all() and gx[rest].isfinite().all()


@pytest.mark.parametrize("dtype,M,F", [(torch.bfloat16, 70, 8), (torch.float32, 70, 8), (torch.float32, 2000, 1100)])
def test_slopes_of_gelu_tanh_far_out(dtype, M, F):
    """1 far above 0 and 0 far below it, where the cube is beyond fp32."""
    K = 132
    far = torch.tensor([1e13, 2e19, 1e20, 1e30, -1e13, -2e19, -1e20, -1e30])
    x = torch.zeros(M, K, dtype=dtype)
    x[:, 0], x[:, 1] = far.repeat(M // 8 + 1)[:M], 1.0
    gate, up = torch.zeros(F, K, dtype=dtype), torch.zeros(F, K, dtype=dtype)
    gate[:, 0], up[:, 1] = 1.0, 1.0
    leaves = [t.to(DEV).requires_grad_() for t in (x, gate, up)]
    h = gated_linear(*leaves, activation="gelu_tanh")
    (gx,) = torch.autograd.grad(h, leaves[:1], torch.ones_like(h))
    assert torch.equal(h, leaves[0][:, :1].clamp_min(0).expand(M, F))
    assert torch.equal(gx[:, 0], F * (leaves[0][:, 0] > 0).to(dtype))


@pytest.mark.parametrize("M,F", [(70, 8), (2000, 1024)])
def test_slopes_of_the_sigmoid_far_out(M, F):
    """e^-|g| (1 + e^-|g|)^-2 with its own bits either way: the exponential's argument is rounded
    (|g| / ln 2, and twice over: the product and its constant), and so are four more steps."""
    K = 132
    x = torch.zeros(M, K)
    x[:, 0], x[:, 1] = torch.linspace(-60, 60, M), 1.0
    gate, up = torch.zeros(F, K), torch.zeros(F, K)
    gate[:, 0], up[:, 1] = 1.0, 1.0
    leaves = [t.to(DEV).requires_grad_() for t in (x, gate, up)]
    h = gated_linear(*leaves, activation="sigmoid")
    gh = torch.zeros_like(h)
    gh[:, 0] = 1.0  # one term a sum
    (gx,) = torch.autograd.grad(h, leaves[:1], gh)
    g = x[:, 0].double()
    e = torch.exp(-g.abs())
    want = e / (1 + e) ** 2
    off = (gx[:, 0].double().cpu() - want).abs() / want
    assert (off <= (2 * g.abs() + 16) * 2.0 ** -23).all(), float(off.max())
    assert ((h[:, 0].double().cpu() - torch.sigmoid(g)).abs() <= (2 * g.abs() + 16) * 2.0 ** -23 * torch.sigmoid(g)).all()

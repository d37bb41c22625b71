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

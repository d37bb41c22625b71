"""The gated projections' sums over long contractions in fp32: no chain of more than 512
products, however long the sum."""
from __future__ import annotations

import pytest
import torch

from neural_shift_cuda import gated_linear

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda"
LONG = 8192


def close(got, want):
    """512 products in a row, then a chain of such sums (of 480 in the smallest tiles); each addition
    rounds or cuts off a step of 2^-23 of what is there, which is at most `want`.  (In one chain the
    8191 quarters behind 2^24 would all be lost: 2048, against 1060.)"""
    off = (got.double().cpu() - want).abs().max()
    assert off <= (512 + LONG // 480 + 1) * 2.0 ** -23 * want, float(off)


def line():
    x = torch.full((LONG,), 0.25)
    x[0] = 2.0 ** 24
    return x, float(x.double().sum())


@pytest.mark.parametrize("M", [70, 300])
def test_values(M):
    x, want = line()
    gate, up = torch.zeros(40, LONG), torch.ones(40, LONG)
    gate[:, 0] = 2.0 ** -24
    h = gated_linear(x.expand(M, LONG).contiguous().to(DEV), gate.to(DEV), up.to(DEV), activation="relu")
    close(h, want)


@pytest.mark.parametrize("name", ["gate", "up"])
def test_the_weights_gradients(name):
    x = torch.ones(LONG, 8)
    x[:, 1], want = line()
    w = torch.zeros(40, 8)
    w[:, 0] = 1.0
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, w.clone())]
    h = gated_linear(*leaves, activation="relu")
    grad = torch.autograd.grad(h, leaves[1 if name == "gate" else 2], torch.ones_like(h))[0]
    close(grad[:, 1], want)

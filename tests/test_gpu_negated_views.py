"""Real tensors whose numbers lie in memory with the other sign (a conjugate's imaginary
part), in every place that an operator takes one."""
from __future__ import annotations

import pytest
import torch

from neural_shift_cuda import (biased_attention, gated_linear, layer_norm, qk_norm_rotary, relative_buckets,
                               relative_position_bias, rotary_table)

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda"


def normal(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(DEV)


def negated(t):
    """t's numbers, held as -t."""
    v = torch._neg_view(-t)
    assert v.is_neg() and v.is_contiguous() and torch.equal(v, t)
    return v


def rotary(q, k, wq, wk):
    cos, sin = (t.to(DEV) for t in rotary_table(16, 32))
    return qk_norm_rotary(q, k, wq, wk, cos, sin)


def attention(q, k, v, table):
    return biased_attention(q, k, v, bias_table=table, buckets=relative_buckets(8, 16).to(DEV), causal=True)


CALLS = {
    "norm": (lambda: [normal(6, 40), normal(40), normal(40), normal(6, 40, seed=1)],
             lambda x, w, b, r: layer_norm(x, w, b, residual=r)),
    "norm of one column": (lambda: [normal(6, 1), normal(1), normal(1, seed=1)], layer_norm),
    "gated": (lambda: [normal(6, 40), normal(24, 40), normal(24, 40, seed=1)], gated_linear),
    "rotary": (lambda: [normal(2, 3, 16, 32), normal(2, 1, 16, 32), normal(32), normal(32, seed=1)], rotary),
    "bias": (lambda: [normal(8, 3)],
             lambda t: relative_position_bias(t, relative_buckets(8, 16).to(DEV), 9, 9)),
    "attention": (lambda: [normal(2, 3, 16, 32), normal(2, 1, 16, 32), normal(2, 1, 16, 32, seed=1), normal(8, 3)],
                  attention),
}


def outputs(f, leaves):
    out = f(*leaves)
    return out if isinstance(out, tuple) else (out,)


@pytest.mark.parametrize("name", list(CALLS))
def test_inputs(name):
    make, f = CALLS[name]
    leaves = make()
    want = outputs(f, leaves)
    for i in range(len(leaves)):
        given = [negated(t) if i == j else t for j, t in enumerate(leaves)]
        for a, b in zip(outputs(f, given), want):
            assert torch.equal(a, b), f"argument {i}"


@pytest.mark.parametrize("name", list(CALLS))
def test_gradients(name):
    make, f = CALLS[name]
    leaves = [t.requires_grad_() for t in make()]
    want = outputs(f, leaves)
    ups = [normal(*o.shape, seed=7) for o in want]
    grads = torch.autograd.grad(want, leaves, ups, retain_graph=True)
    for a, b in zip(torch.autograd.grad(want, leaves, [negated(u) for u in ups]), grads):
        assert torch.equal(a, b), "upstream"
    for i in range(len(leaves)):
        given = [negated(t.detach()).requires_grad_() if i == j else t for j, t in enumerate(leaves)]
        out = outputs(f, given)
        for a, b in zip((*out, *torch.autograd.grad(out, given, ups)), (*want, *grads)):
            assert torch.equal(a, b), f"argument {i}"

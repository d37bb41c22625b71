"""The token operators under torch.jit.trace and forward-mode differentiation: a
trace runs the kernels again, and a tangent is refused, not dropped."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from neural_shift_cuda import biased_attention
from test_gpu_token_calls import DEV, calls, tensors

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


def other(leaves):
    return [t.flip(0) * 0.5 + 0.25 for t in leaves]


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("name", ["attention", "norm", "bias"])
def test_a_trace_runs_the_kernels(name, train):
    leaves, f = calls()[name]
    leaves = [t.requires_grad_(train) for t in leaves]
    traced = torch.jit.trace(lambda *t: f(*t) * 2.0, leaves)
    for _ in range(2):
        leaves = [t.detach().requires_grad_(train) for t in other(leaves)]
        want, got = f(*leaves) * 2.0, traced(*leaves)
        assert torch.equal(got, want)
        if train:
            ups = torch.ones_like(want)
            for a, b in zip(torch.autograd.grad(got, leaves, ups),
                            torch.autograd.grad(want, leaves, ups)):
                assert torch.equal(a, b)


def test_a_traced_call_with_masks_and_degree():
    q, k, v = tensors((2, 2, 30, 16), (2, 2, 40, 16), (2, 2, 40, 16))
    lengths = torch.tensor([40, 33], device=DEV)

    def f(q, k, v, lengths):
        out, degree = biased_attention(q, k, v, causal=True, cap=9.0, lengths=lengths,
                                       return_log_degree=True)
        return out + degree[..., None]

    traced = torch.jit.trace(f, (q, k, v, lengths))
    lengths = torch.tensor([31, 40], device=DEV)
    assert torch.equal(traced(k[:, :, :30], q.new_ones(k.shape), v, lengths),
                       f(k[:, :, :30], q.new_ones(k.shape), v, lengths))


@pytest.mark.parametrize("trains", [False, True])
@pytest.mark.parametrize("name", ["attention", "norm", "bias"])
def test_tangents_are_refused(name, trains):
    leaves, f = calls()[name]
    for n in range(len(leaves)):
        with forward_ad.dual_level():
            given = [t.detach().clone().requires_grad_(trains) for t in leaves]
            given[n] = forward_ad.make_dual(given[n], torch.ones_like(given[n]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(*given)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                f(*given)
    f(*leaves)  # and none is left behind

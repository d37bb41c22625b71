"""The token operators' autograd nodes: which gradients are formed, when they
are refused, and on which stream."""
from __future__ import annotations

import pytest
import torch

from neural_shift_cuda import (biased_attention, qk_norm_rotary, relative_buckets,
                               relative_position_bias, rotary_table)

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda"


def tensors(*shapes, dtype=torch.float32):
    g = torch.Generator().manual_seed(3)
    return [torch.randn(*s, generator=g).to(DEV, dtype) for s in shapes]


@pytest.mark.parametrize("have", ["both", "q", "k"])
@pytest.mark.parametrize("train", ["all", "k weight", "q weight", "q"])
def test_norm_gradients_go_to_their_inputs(have, train):
    """With one weight missing the other's gradient is still its own."""
    q, k, wq, wk, go = tensors((2, 3, 5, 16), (2, 2, 5, 16), (16,), (16,), (2, 3, 5, 16))
    wq, wk = (wq if have != "k" else None), (wk if have != "q" else None)
    cos, sin = (t.to(DEV) for t in rotary_table(5, 8))
    leaves = {"q": q, "k": k, "q weight": wq, "k weight": wk}
    want = {n for n, t in leaves.items() if t is not None and train in ("all", n)}
    if not want:
        pytest.skip("the weight that trains is not there")
    for n in want:
        leaves[n].requires_grad_()

    def run(on):
        a = [None if t is None else t.detach().to(on).requires_grad_(t.requires_grad)
             for t in leaves.values()]
        yq, yk = qk_norm_rotary(*a, cos.to(on), sin.to(on))
        loss = (yq * go.to(on)).sum() + yk.square().sum() + yk.sum()
        loss.backward()
        return [None if t is None else t.grad for t in a]

    for n, got, ref in zip(leaves, run(DEV), run("cpu")):
        assert (got is None) == (ref is None) == (n not in want), n
        if got is not None:
            torch.testing.assert_close(got.cpu(), ref, rtol=1e-4, atol=1e-4)


def calls():
    q, k, v, table = tensors((1, 2, 40, 16), (1, 2, 40, 16), (1, 2, 40, 16), (8, 2))
    buckets = relative_buckets(8, 20).to(DEV)
    cos, sin = (t.to(DEV) for t in rotary_table(40, 16))
    return {
        "attention": ([q, k, v, table], lambda q, k, v, t: biased_attention(
            q, k, v, bias_table=t, buckets=buckets)),
        "norm": ([q, k], lambda q, k: qk_norm_rotary(q, k, None, None, cos, sin)[0]),
        "bias": ([table], lambda t: relative_position_bias(t, buckets, 30, 40)),
    }


@pytest.mark.parametrize("name", ["attention", "norm", "bias"])
def test_no_gradient_of_a_gradient(name):
    leaves, f = calls()[name]
    leaves = [t.requires_grad_() for t in leaves]
    grads = torch.autograd.grad(f(*leaves).square().sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        sum(g.square().sum() for g in grads).backward()


@pytest.mark.parametrize("name", ["attention", "norm", "bias"])
def test_backward_twice_gives_the_same_bits(name):
    leaves, f = calls()[name]
    leaves = [t.requires_grad_() for t in leaves]
    out = f(*leaves)
    go = torch.ones_like(out)
    first = torch.autograd.grad(out, leaves, go, retain_graph=True)
    again = torch.autograd.grad(out, leaves, go)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, leaves, go)


@pytest.mark.parametrize("name", ["attention", "norm"])
def test_a_changed_input_is_noticed(name):
    leaves, f = calls()[name]
    bases = [t.requires_grad_() for t in leaves]
    leaves = [t * 1.0 for t in bases]
    out = f(*leaves)
    leaves[1].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("name", ["attention", "norm", "bias"])
def test_on_another_stream(name):
    leaves, f = calls()[name]
    leaves = [t.requires_grad_() for t in leaves]
    out = f(*leaves)
    want = [out, *torch.autograd.grad(out.square().sum(), leaves)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f(*leaves)
        got = [got, *torch.autograd.grad(got.square().sum(), leaves)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("name", ["attention", "norm", "bias"])
def test_saved_tensors_may_be_kept_elsewhere(name):
    """Hooks that keep a copy on the host."""
    leaves, f = calls()[name]
    leaves = [t.requires_grad_() for t in leaves]
    want = torch.autograd.grad(f(*leaves).square().sum(), leaves)
    with torch.autograd.graph.save_on_cpu():
        out = f(*leaves)
    got = torch.autograd.grad(out.square().sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_one_gradient_of_the_degree_alone():
    q, k, v = (t.requires_grad_() for t in calls()["attention"][0][:3])
    _, degree = biased_attention(q, k, v, return_log_degree=True)
    grads = torch.autograd.grad(degree.sum(), [q, k, v], allow_unused=True)
    ref = [t.detach().cpu().requires_grad_() for t in (q, k, v)]
    _, d = biased_attention(*ref, return_log_degree=True)
    want = torch.autograd.grad(d.sum(), ref, allow_unused=True)
    for a, b in zip(grads, want):
        b = torch.zeros_like(ref[2]) if b is None else b
        torch.testing.assert_close(a.cpu(), b, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("name", ["attention", "norm", "bias"])
def test_double_precision_is_refused(name):
    leaves, f = calls()[name]
    with pytest.raises(RuntimeError, match="not implemented"):
        f(*(t.double() for t in leaves))


def test_refusals_on_the_gpu_are_the_checks_own():
    q, k, v, table = calls()["attention"][0]
    buckets = relative_buckets(8, 20).to(DEV)
    for error, match, f in (
            (ValueError, "multiple of the", lambda: biased_attention(q[:, :1], k, v)),
            (ValueError, "prefix needs causal", lambda: biased_attention(
                q, k, v, prefix=torch.zeros(1, dtype=torch.int32, device=DEV))),
            (ValueError, "buckets come with", lambda: biased_attention(q, k, v, buckets=buckets)),
            (ValueError, "finite", lambda: biased_attention(q, k, v, cap=float("nan"))),
            (ValueError, "buckets must be", lambda: biased_attention(q, k, v, bias_table=table)),
            (ValueError, "lengths must be", lambda: biased_attention(
                q, k, v, lengths=torch.zeros(2, dtype=torch.int32, device=DEV))),
            (ValueError, "lengths must be on", lambda: biased_attention(
                q, k, v, lengths=torch.zeros(1, dtype=torch.int32))),
            (TypeError, "must hold integers", lambda: biased_attention(
                q, k, v, lengths=torch.zeros(1, device=DEV))),
            (ValueError, "must not be negative", lambda: relative_position_bias(
                table, buckets, -1, 3)),
            (ValueError, "buckets must be", lambda: relative_position_bias(table, None, 3, 3)),
            (ValueError, "rows for", lambda: qk_norm_rotary(
                q, k, None, None, torch.ones(3, 4, device=DEV), torch.ones(3, 4, device=DEV))),
            (ValueError, "half", lambda: qk_norm_rotary(
                q, k, None, None, torch.ones(40, 9, device=DEV), torch.ones(40, 9, device=DEV)))):
        with pytest.raises(error, match=match):
            f()


def test_converted_arguments_give_the_same():
    """Masks in 64 bits, tables in double precision, a strided map: the same bits
    as in the kernels' own types."""
    q, k, v, table = calls()["attention"][0]
    buckets = relative_buckets(8, 20).to(DEV)
    docs = (torch.arange(40, device=DEV) // 15)[None]
    lengths = torch.tensor([33], device=DEV)
    slopes = torch.rand(2, device=DEV)
    a = biased_attention(q, k, v, causal=True, documents=docs.int(), lengths=lengths.int(),
                         slopes=slopes, bias_table=table, buckets=buckets)
    b = biased_attention(q, k, v, causal=True, documents=docs, lengths=lengths,
                         slopes=slopes.double(), bias_table=table,
                         buckets=buckets.long().repeat_interleave(2)[::2])
    assert torch.equal(a, b)
    cos, sin = (t.to(DEV) for t in rotary_table(60, 16))
    at = torch.arange(40, device=DEV) + 7
    a = qk_norm_rotary(q, k, None, None, cos, sin, at.int())
    b = qk_norm_rotary(q, k, None, None, cos.double(), sin.double(), at)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.equal(relative_position_bias(table, buckets, 30, 40),
                       relative_position_bias(table, buckets.long(), 30, 40))

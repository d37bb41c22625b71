"""Sound data stay on the tiles: the computation pair by pair, for rows that end
in an infinity or a NaN, takes some fifty times as long, so a call that reaches
it shows in its time next to a like one that does not."""
from __future__ import annotations

import pytest
import torch

import token_dense as dense
from neural_shift_cuda import biased_attention, relative_buckets

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda:0"


def tensors(L, dtype, D=64):
    g = torch.Generator(device=DEV).manual_seed(L)
    return [torch.randn(1, 8, L, D, generator=g, device=DEV).to(dtype) for _ in range(4)]


def step(q, k, v, go, **rules):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = biased_attention(*leaves, **rules)
    return [out.detach(), *torch.autograd.grad(out, leaves, go)]


def time_of(f):
    f()
    best = float("inf")
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        f()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


def alike(first, second):
    slow, fast = time_of(first), time_of(second)
    print(f"{slow:.3f} ms, {fast:.3f} ms")
    assert slow <= 5 * fast


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_a_scale_of_zero(dtype, D):
    """Every visible key weighs the same; a masked score is not 0 times infinity."""
    L = 2050
    q, k, v, go = tensors(L, dtype, D)
    alike(lambda: step(q, k, v, go, causal=True, scale=0.0),
          lambda: step(q, k, v, go, causal=True, scale=0.125))
    q, k, v, go = (t[:, :1, :300].contiguous() for t in (q, k, v, go))
    got, want = step(q, k, v, go, causal=True, scale=0.0), dense.attention(q, k, v, go, causal=True, scale=0.0)
    u = torch.finfo(dtype).eps / 2
    for n, g in zip(("out", "gq", "gk", "gv"), got):
        assert (g.double() - want[n]).norm() <= (2 * u + 2.0 ** -18) * want[n].norm(), n


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
def test_a_large_bias(dtype, D):
    """e^100 is beyond fp32; rows past the queries' end have no maximum to take off."""
    q, k, v, go = tensors(2050, dtype, D)
    buckets = relative_buckets(8, 20, device=DEV)
    table = torch.zeros(8, 8, device=DEV).to(dtype)
    alike(lambda: step(q, k, v, go, bias_table=table + 100, buckets=buckets),
          lambda: step(q, k, v, go, bias_table=table, buckets=buckets))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cap", [None, 40.0])
def test_large_upstream_gradients(cap, D):
    """dx beyond fp16's largest number."""
    q, k, v, go = tensors(2050, torch.float16, D)
    alike(lambda: step(q * 4, k * 4, v * 64, go * 1024, scale=2.0 / D, cap=cap),
          lambda: step(q * 4, k * 4, v, go, scale=2.0 / D, cap=cap))

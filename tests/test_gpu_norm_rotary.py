"""qk_norm_rotary and relative_position_bias on the GPU against the formulas in
64 bits."""
from __future__ import annotations

import pytest
import torch

import token_oracle as oracle
from neural_shift_cuda import (qk_norm_rotary, relative_buckets, relative_position_bias,
                               rotary_table)

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def norm_check(B, Hq, Hk, L, D, rot, dtype, interleaved=False, weights=True, positions=None,
               layout=lambda t: t.to(DEV), seed=0):
    g = torch.Generator().manual_seed(seed)
    dt = TYPES[dtype]
    q, gq = (torch.randn(B, Hq, L, D, generator=g).to(dt) for _ in range(2))
    k, gk = (torch.randn(B, Hk, L, D, generator=g).to(dt) for _ in range(2))
    wq, wk = (torch.randn(D, generator=g).to(dt) if weights else None for _ in range(2))
    cos, sin = rotary_table(500, rot)
    at = torch.randint(0, 500, (B, L), generator=g) if positions is None else positions
    qd, kd = layout(q).requires_grad_(), layout(k).requires_grad_()
    ws = [None if w is None else w.to(DEV).requires_grad_() for w in (wq, wk)]
    out = qk_norm_rotary(qd, kd, *ws, cos.to(DEV), sin.to(DEV), at.to(DEV), eps=1e-6,
                         interleaved=interleaved)
    leaves = [qd, kd] + [w for w in ws if w is not None]
    grads = torch.autograd.grad(out, leaves, [layout(gq), layout(gk)], allow_unused=True)
    at = at.expand(B, L)
    for n, (x, w, up) in enumerate(((q, wq, gq), (k, wk, gk))):
        if not x.numel():
            continue
        vals, tols = oracle.norm_rotary(x, w, cos, sin, at, 1e-6, interleaved, up)
        oracle.close(out[n], vals["out"], tols["out"], f"out {n}")
        oracle.close(grads[n], vals["gx"], tols["gx"], f"gx {n}")
        if weights:
            oracle.close(grads[2 + n], vals["gw"], tols["gw"], f"gw {n}")
        with torch.no_grad():
            again = qk_norm_rotary(qd, kd, *ws, cos.to(DEV), sin.to(DEV), at.to(DEV), eps=1e-6,
                                   interleaved=interleaved)[n]
            torch.testing.assert_close(again, out[n].detach(), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(128, 128), (64, 32), (80, 40), (96, 96), (256, 64), (16, 16),
                                   (50, 20), (7, 6), (512, 512), (1, 0), (72, 8)])
def test_widths(dtype, interleaved, D, rot):
    norm_check(2, 3, 2, 5, D, rot, dtype, interleaved)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("B,Hq,Hk,L", [(1, 1, 1, 1), (8, 8, 2, 1), (1, 5, 5, 77), (3, 4, 0, 9),
                                       (2, 0, 3, 4)])
def test_shapes(dtype, B, Hq, Hk, L):
    norm_check(B, Hq, Hk, L, 64, 64, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_layouts(dtype):
    norm_check(2, 4, 2, 6, 64, 64, dtype,
               layout=lambda t: t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2).detach())
    norm_check(2, 4, 2, 6, 64, 64, dtype,
               layout=lambda t: torch.nn.functional.pad(t, (1, 2)).to(DEV)[..., 1:65].detach())
    norm_check(2, 4, 2, 6, 64, 64, dtype,
               layout=lambda t: t.transpose(2, 3).contiguous().to(DEV).transpose(2, 3).detach())
    norm_check(2, 4, 2, 6, 64, 64, dtype, weights=False)


def test_positions():
    norm_check(2, 2, 2, 5, 64, 64, "fp32", positions=torch.tensor([0, 499, 3, 3, 250]))
    # outside the table: NaN, and nothing is read
    norm_check(2, 2, 2, 5, 64, 32, "bf16",
               positions=torch.tensor([[0, -1, 3, 500, 1], [1 << 40, 2, -(1 << 40), 4, 499]]))


def test_many_rows():
    """More rows than the workgroups of one turn, odd in number."""
    g = torch.Generator().manual_seed(0)
    q = torch.randn(3, 1027, 16, 64, generator=g, dtype=torch.float32).to(DEV).transpose(1, 2)
    k = torch.randn(3, 1027, 5, 64, generator=g, dtype=torch.float32).to(DEV).transpose(1, 2)
    w = torch.ones(64, device=DEV)
    cos, sin = rotary_table(1027, 64, device=DEV)
    ls = [t.detach().requires_grad_() for t in (q, k, w)]
    out = qk_norm_rotary(ls[0], ls[1], ls[2], ls[2], cos, sin)
    up = [torch.randn(o.shape, generator=g).to(DEV) for o in out]
    grads = torch.autograd.grad(out, ls, up)
    dl = [t.detach().double().requires_grad_() for t in (q, k, w)]
    res = []
    for x in dl[:2]:
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * dl[2]
        a, b = y[..., :32], y[..., 32:]
        c, s = cos.double(), sin.double()
        res.append(torch.cat((a * c - b * s, a * s + b * c), -1))
    want = torch.autograd.grad(res, dl, [u.double() for u in up])
    for o, r in zip(out, res):
        assert float((o - r).detach().abs().max()) < 80 * oracle.F32 * float(r.detach().abs().max())
    for n in range(2):
        assert float((grads[n].double() - want[n]).abs().max()) < 240 * oracle.F32 * 20
    # rows * terms of about 1, summed in runs: their magnitudes' sum times the longest chain
    rows = 3 * 1027 * 21
    assert float((grads[2].double() - want[2]).abs().max()) < 512 * oracle.F32 * rows


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("Lq,Lk,reach", [(1, 1, 0), (1, 70, 5), (33, 33, 10), (70, 131, 64),
                                         (65, 40, 8), (10, 300, 2000), (130, 77, 1)])
def test_position_bias(dtype, Lq, Lk, reach):
    g = torch.Generator().manual_seed(1)
    dt = TYPES[dtype]
    buckets = torch.randint(0, 11, (2 * reach + 1,), generator=g)
    table = torch.randn(11, 3, generator=g).to(dt)
    t = table.to(DEV).requires_grad_()
    out = relative_position_bias(t, buckets.to(DEV), Lq, Lk)
    assert out.dtype == dt
    assert torch.equal(out.double().cpu(), oracle.position_bias(table, buckets, Lq, Lk))
    go = torch.randn(3, Lq, Lk, generator=g).to(dt)
    (grad,) = torch.autograd.grad(out, t, go.to(DEV))
    want, tol = oracle.position_bias_grad(go, buckets, 11)
    oracle.close(grad, want, tol, "grad")
    (again,) = torch.autograd.grad(relative_position_bias(t, buckets.to(DEV), Lq, Lk), t,
                                   go.to(DEV))
    assert torch.equal(grad, again)


def test_position_bias_large():
    g = torch.Generator(device=DEV).manual_seed(1)
    buckets = relative_buckets(32, 128, device=DEV)
    table = torch.randn(32, 5, generator=g, device=DEV).requires_grad_()
    out = relative_position_bias(table, buckets, 1000, 1503)
    rel = (torch.arange(1503, device=DEV) - (torch.arange(1000, device=DEV)[:, None] + 503))
    ids = buckets.long()[rel.clamp(-128, 128) + 128]
    assert torch.equal(out, table.detach()[ids].permute(2, 0, 1))
    go = torch.randn(out.shape, generator=g, device=DEV)
    (grad,) = torch.autograd.grad(out, table, go)
    for b in range(32):
        at = go.double() * (ids == b)
        # the longest chain of additions: a lane's part of the far ends
        tol = 700 * oracle.F32 * at.abs().sum((1, 2))
        assert ((grad[b].double() - at.sum((1, 2))).abs() <= tol).all()


def test_position_bias_bad_buckets():
    """A bucket the table lacks: NaN where it is used, nothing read, no gradient."""
    table = torch.randn(4, 2, device=DEV).requires_grad_()
    buckets = torch.tensor([0, 7, -1, 1, 1 << 30], device=DEV)
    out = relative_position_bias(table, buckets, 3, 3)
    want = oracle.position_bias(table.detach().cpu(), buckets.cpu(), 3, 3)
    oracle.close(out, want, torch.zeros(()), "bias")
    (grad,) = torch.autograd.grad(out, table, torch.ones_like(out))
    assert torch.equal(grad.cpu(), oracle.position_bias_grad(
        torch.ones(2, 3, 3), buckets.cpu(), 4)[0].float())


def test_position_bias_empty():
    table = torch.randn(4, 2, device=DEV).requires_grad_()
    out = relative_position_bias(table, relative_buckets(4, 8, device=DEV), 0, 7)
    assert out.shape == (2, 0, 7)
    assert not torch.autograd.grad(out.sum(), table)[0].any()


def test_captured_step():
    """Norm, bias and their gradients in a graph, replayed with new inputs."""
    g = torch.Generator().manual_seed(2)
    q = torch.randn(2, 4, 33, 64, generator=g).to(DEV)
    k = torch.randn(2, 2, 33, 64, generator=g).to(DEV)
    w = torch.randn(64, generator=g).to(DEV)
    table = torch.randn(8, 4, generator=g).to(DEV)
    buckets = relative_buckets(8, 16, device=DEV)
    cos, sin = rotary_table(33, 64, device=DEV)
    static = [q, k, w, table]

    def step(ts):
        ls = [t.detach().requires_grad_() for t in ts]
        a, b = qk_norm_rotary(ls[0], ls[1], ls[2], ls[2], cos, sin)
        c = relative_position_bias(ls[3], buckets, 33, 33)
        grads = torch.autograd.grad([a, b, c], ls, [a.detach() + 1, b.detach() + 1, c.detach()])
        return [a.detach(), b.detach(), c.detach(), *grads]

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(static)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(static)
    for r in range(4):
        new = [torch.randn(t.shape, generator=g).to(DEV) for t in static]
        want = step(new)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(res, want)), f"replay {r}"

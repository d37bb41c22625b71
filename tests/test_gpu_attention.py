"""biased_attention on the GPU against the formulas in 64 bits: values, log
degrees and every gradient, at the lengths, masks, biases, types and strides
where tiles, tails and empty rows meet."""
from __future__ import annotations

import pytest
import torch

import token_oracle as oracle
from neural_shift_cuda import biased_attention, relative_buckets

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def inputs(B, Hq, Hk, Lq, Lk, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    dt = TYPES[dtype]
    q = torch.randn(B, Hq, Lq, D, generator=g).to(dt)
    k = torch.randn(B, Hk, Lk, D, generator=g).to(dt)
    v = torch.randn(B, Hk, Lk, D, generator=g).to(dt)
    return q, k, v, torch.randn(B, Hq, Lq, D, generator=g).to(dt), g


def on_gpu(rules):
    return {n: x.to(DEV) if isinstance(x, torch.Tensor) else x for n, x in rules.items()}


def check(q, k, v, go, rules, gdegree=None, layout=lambda t: t.to(DEV)):
    vals, tols = oracle.attention(q, k, v, go=go, gdegree=gdegree, **rules)
    qd, kd, vd = (layout(t).requires_grad_() for t in (q, k, v))
    r = on_gpu(rules)
    leaves = {"gq": qd, "gk": kd, "gv": vd}
    if "bias_table" in r:
        leaves["gtable"] = r["bias_table"].requires_grad_()
    out, degree = biased_attention(qd, kd, vd, return_log_degree=True, **r)
    ups = [layout(go)] + ([gdegree.to(DEV)] if gdegree is not None else [])
    grads = torch.autograd.grad([out, degree][:len(ups)], list(leaves.values()), ups)
    oracle.close(out, vals["out"], tols["out"], "out")
    oracle.close(degree, vals["degree"], tols["degree"], "degree")
    for n, g in zip(leaves, grads):
        oracle.close(g, vals[n], tols[n], n)
    with torch.no_grad():  # without gradients, and without the degree
        again = biased_attention(qd, kd, vd, **r)
    oracle.close(again, vals["out"], tols["out"], "out of a forward alone")
    return out, grads


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 67), (63, 65), (130, 130), (129, 257), (200, 64)])
def test_lengths(dtype, Lq, Lk):
    q, k, v, go, _ = inputs(2, 2, 1, Lq, Lk, 64, dtype)
    check(q, k, v, go, {"causal": True})
    check(q, k, v, go, {})


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D", [8, 24, 40, 64, 72, 96, 112, 128, 20, 1])
def test_widths(dtype, D):
    q, k, v, go, _ = inputs(1, 4, 2, 90, 150, D, dtype)
    check(q, k, v, go, {"cap": 3.0, "causal": True})


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("cap,scale", [(50.0, None), (2.0, 1.0), (30.0, -0.5), (1e4, 0.2)])
def test_caps_and_scales(dtype, cap, scale):
    q, k, v, go, _ = inputs(1, 2, 2, 70, 140, 64, dtype)
    check(q, k, v, go, {"cap": cap, "scale": scale})


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("heads", [(1, 1), (6, 2), (8, 1), (5, 5), (34, 2)])
def test_head_groups(dtype, heads):
    q, k, v, go, _ = inputs(2, *heads, 33, 70, 32, dtype)
    check(q, k, v, go, {"causal": True, "cap": 10.0})


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("Lq", [150, 1])
def test_slopes(dtype, Lq):
    q, k, v, go, _ = inputs(2, 4, 2, Lq, 290, 64, dtype)
    slopes = torch.tensor([0.5, 0.1, 0.0, 0.01])
    check(q, k, v, go, {"slopes": slopes})
    check(q, k, v, go, {"slopes": slopes, "causal": True, "cap": 20.0})


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("Lq,Lk,reach", [(200, 200, 20), (70, 333, 100), (1, 90, 7), (150, 150, 1),
                                         (333, 333, 400), (65, 130, 0)])
def test_bucketed_bias(dtype, Lq, Lk, reach):
    q, k, v, go, g = inputs(2, 4, 2, Lq, Lk, 40, dtype)
    buckets = torch.randint(0, 9, (2 * reach + 1,), generator=g, dtype=torch.int32)
    table = torch.randn(9, 4, generator=g).to(q.dtype)
    check(q, k, v, go, {"bias_table": table, "buckets": buckets})
    check(q, k, v, go, {"bias_table": table, "buckets": buckets, "causal": True, "cap": 5.0,
                        "slopes": torch.tensor([0.2, 0.0, 0.02, 0.1])})


def test_bias_that_excludes_distances():
    """-inf in the table; the type's lowest value is a score like any other."""
    q, k, v, go, _ = inputs(1, 2, 2, 100, 100, 32, "fp32")
    reach = 10
    buckets = (torch.arange(-reach, reach + 1).abs() >= reach).int()
    table = torch.tensor([[0.3, -0.2], [-float("inf"), 1.0]])
    check(q, k, v, go, {"bias_table": table, "buckets": buckets})
    # a row all of whose scores are the lowest value: even weights
    low = torch.full((2, 2), torch.finfo(torch.float32).min)
    out = biased_attention(q.to(DEV), k.to(DEV), v.to(DEV), bias_table=low.to(DEV),
                           buckets=buckets.to(DEV))
    want = v.double().mean(2, keepdim=True).expand(1, 2, 100, 32)
    oracle.close(out, want, 200 * oracle.F32 * v.double().abs().mean(2, keepdim=True), "even")


def test_every_distance_excluded():
    q, k, v, go, _ = inputs(1, 2, 2, 70, 70, 32, "bf16")
    table = torch.full((1, 2), -float("inf"), dtype=torch.bfloat16)
    buckets = torch.zeros(3, dtype=torch.int32)
    out, grads = check(q, k, v, go, {"bias_table": table, "buckets": buckets})
    assert not out.any() and not any(g.any() for g in grads)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("Lq", [190, 1, 40])
def test_lengths_of_a_cache(dtype, Lq):
    q, k, v, go, _ = inputs(6, 2, 2, Lq, 190, 64, dtype)
    lengths = torch.tensor([190, 0, 1, 64, 129, 500], dtype=torch.int64)
    # what lies behind the filled part is never used
    for b, n in enumerate(lengths.tolist()):
        k[b, :, n:], v[b, :, n:] = float("nan"), float("inf")
    check(q, k, v, go, {"lengths": lengths})
    check(q, k, v, go, {"lengths": lengths, "causal": True, "cap": 9.0})


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("causal", [False, True])
def test_documents(dtype, causal):
    q, k, v, go, g = inputs(3, 2, 1, 300, 300, 32, dtype)
    docs = torch.empty(3, 300, dtype=torch.int32)
    docs[0] = torch.arange(300) // 37
    docs[1] = torch.randint(-1, 4, (300,), generator=g)  # in no order
    docs[2] = 5
    docs[2, 130:] = -1
    k[2, :, 130:], v[2, :, 130:] = float("inf"), float("nan")
    check(q, k, v, go, {"documents": docs, "causal": causal})


def test_documents_of_the_last_queries():
    q, k, v, go, _ = inputs(2, 2, 2, 50, 210, 32, "bf16")
    docs = (torch.arange(210) // 90).int().repeat(2, 1)
    check(q, k, v, go, {"documents": docs, "causal": True,
                        "lengths": torch.tensor([210, 100], dtype=torch.int32)})


@pytest.mark.parametrize("dtype", list(TYPES))
def test_prefix(dtype):
    q, k, v, go, _ = inputs(5, 2, 2, 200, 200, 32, dtype)
    check(q, k, v, go, {"causal": True, "cap": 20.0,
                        "prefix": torch.tensor([0, 1, 70, 200, 1000], dtype=torch.int32)})


def test_prefix_with_more_queries_than_keys():
    q, k, v, go, _ = inputs(2, 2, 2, 200, 90, 32, "fp32")
    check(q, k, v, go, {"causal": True, "prefix": torch.tensor([0, 5], dtype=torch.int32)})


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_gradient_through_the_degree(dtype):
    q, k, v, go, g = inputs(2, 4, 2, 100, 130, 64, dtype)
    check(q, k, v, go, {"causal": True, "cap": 8.0},
          gdegree=torch.randn(2, 4, 100, generator=g))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_layouts(dtype):
    q, k, v, go, _ = inputs(2, 4, 4, 100, 100, 64, dtype)
    rules = {"causal": True}
    # tokens before heads
    out, _ = check(q, k, v, go, rules,
                   layout=lambda t: t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2))
    assert out.transpose(1, 2).is_contiguous()
    # a slice of one projection, rows on 16 bytes
    check(q, k, v, go, rules, layout=lambda t: torch.cat((t, t), -1).to(DEV)[..., 64:].detach())
    # rows off 16 bytes, a stride in the last place
    check(q, k, v, go, rules,
          layout=lambda t: torch.nn.functional.pad(t, (1, 2)).to(DEV)[..., 1:65].detach())
    check(q, k, v, go, rules, layout=lambda t: t.transpose(2, 3).contiguous().to(DEV).transpose(2, 3))


def test_broadcast_keys():
    q, k, v, go, _ = inputs(1, 2, 2, 60, 60, 32, "fp32")
    qd = q.expand(3, 2, 60, 32)
    kd, vd = k[:, :1].to(DEV).requires_grad_(), v[:, :1].to(DEV).requires_grad_()
    out = biased_attention(qd.to(DEV), kd.expand(3, 2, 60, 32), vd.expand(3, 2, 60, 32))
    gk, gv = torch.autograd.grad(out, (kd, vd), go.to(DEV).expand(3, 2, 60, 32))
    vals, tols = oracle.attention(qd, k[:, :1].expand(3, 2, 60, 32), v[:, :1].expand(3, 2, 60, 32),
                                  go=go.expand(3, 2, 60, 32))
    for got, n in ((gk, "gk"), (gv, "gv")):
        oracle.close(got, vals[n].sum((0, 1), keepdim=True), 2 * tols[n].sum((0, 1), keepdim=True), n)


def test_same_bits_again():
    q, k, v, go, g = inputs(2, 4, 2, 300, 300, 64, "bf16")
    table = torch.randn(16, 4, generator=g).bfloat16().to(DEV).requires_grad_()
    buckets = relative_buckets(16, 100, device=DEV)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)] + [table]
    runs = []
    for _ in range(3):
        out = biased_attention(*leaves[:3], cap=30.0, bias_table=table, buckets=buckets)
        runs.append([out.detach(), *torch.autograd.grad(out, leaves, go.to(DEV))])
    for other in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(runs[0], other))


def test_empty_calls():
    for shape in ((0, 2, 5, 32), (2, 0, 5, 32), (2, 2, 0, 32)):
        q = torch.randn(shape, device=DEV).requires_grad_()
        k = torch.randn(shape[0], shape[1], 5, 32, device=DEV).requires_grad_()
        out, degree = biased_attention(q, k, k, return_log_degree=True)
        assert out.shape == shape and degree.shape == shape[:3]
        gq, gk = torch.autograd.grad(out.sum(), (q, k))
        assert gq.shape == q.shape and gk.shape == k.shape and not gk.any()
    q = torch.randn(1, 2, 5, 32, device=DEV).requires_grad_()
    k = torch.randn(1, 2, 0, 32, device=DEV)
    out, degree = biased_attention(q, k, k, return_log_degree=True)
    assert not out.any() and (degree == -float("inf")).all()
    assert not torch.autograd.grad(out.sum(), q)[0].any()


def test_differences():
    """The gradient against central differences of the forward in fp32."""
    q, k, v, go, _ = inputs(1, 2, 1, 12, 20, 16, "fp32")
    buckets = relative_buckets(8, 10, device=DEV)
    table = torch.randn(8, 2, generator=torch.Generator().manual_seed(3)).to(DEV)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)] + [table.requires_grad_()]

    def f(*t):
        out, deg = biased_attention(*t[:3], cap=4.0, bias_table=t[3], buckets=buckets,
                                    return_log_degree=True)
        return (out * go.to(DEV)).double().sum() + (deg.double() * 0.3).sum()

    grads = torch.autograd.grad(f(*leaves), leaves)
    gen = torch.Generator().manual_seed(5)
    for n, (x, g) in enumerate(zip(leaves, grads)):
        d = torch.randn(x.shape, generator=gen).to(DEV)
        h = 2.0 ** -7
        with torch.no_grad():
            up = f(*[t + h * d if m == n else t for m, t in enumerate(leaves)])
            down = f(*[t - h * d if m == n else t for m, t in enumerate(leaves)])
        # third derivatives times h^2 / 6, and fp32's error over 2 h
        want, got = float((up - down) / (2 * h)), float((g.double() * d.double()).sum())
        assert abs(want - got) <= 2e-3 * float((g.abs().double() * d.abs().double()).sum()) + 1e-3


def test_other_streams():
    q, k, v, go, _ = inputs(2, 4, 2, 200, 200, 64, "bf16")
    vals, tols = oracle.attention(q, k, v, go=go, causal=True)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        out = biased_attention(*leaves, causal=True)
        grads = torch.autograd.grad(out, leaves, go.to(DEV))
    st.synchronize()
    oracle.close(out, vals["out"], tols["out"], "out")
    for n, g in zip(("gq", "gk", "gv"), grads):
        oracle.close(g, vals[n], tols[n], n)


def test_captured_forward_and_backward():
    """A graph of a whole step, replayed with new inputs between eager work."""
    q, k, v, go, g = inputs(2, 4, 2, 130, 130, 64, "bf16")
    table = torch.randn(16, 4, generator=g).bfloat16()
    buckets = relative_buckets(16, 50, device=DEV)
    static = [t.to(DEV) for t in (q, k, v, table, go)]

    def step(ts):
        leaves = [t.detach().requires_grad_() for t in ts[:4]]
        out = biased_attention(*leaves[:3], cap=20.0, causal=True, bias_table=leaves[3],
                               buckets=buckets)
        return [out.detach(), *torch.autograd.grad(out, leaves, ts[4])]

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(static)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(static)
    for r in range(4):
        new = [torch.randn(t.shape, generator=g).to(t.dtype).to(DEV) for t in static]
        want = step(new)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(res, want)), f"replay {r}"

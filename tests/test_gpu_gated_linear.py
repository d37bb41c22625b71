"""gated_linear on the GPU against its formulas in 64 bits."""
from __future__ import annotations

import pytest
import torch

import block_oracle as oracle
from neural_shift_cuda import gated_linear

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
KINDS = ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]


def inputs(M, K, F, dtype, seed=0, up=1.0):
    g = torch.Generator().manual_seed(seed)
    dt = TYPES[dtype]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=g) * by).to(dt)

    return normal(M, K), normal(F, K, by=K ** -0.5), normal(F, K, by=K ** -0.5), normal(M, F, by=up)


def check(M, K, F, dtype, kind="silu", seed=0, up=1.0, layout=lambda t: t.to(DEV), average=False):
    t = inputs(M, K, F, dtype, seed, up)
    x, gate, upw, gh = (layout(v) for v in t)
    vals, tols = oracle.gated(*t[:3], kind, t[3])
    with torch.no_grad():
        oracle.close(gated_linear(x, gate, upw, activation=kind).view(M, F), vals["h"], tols["h"], "h alone")
    leaf = [v.detach().requires_grad_() for v in (x, gate, upw)]
    h = gated_linear(*leaf, activation=kind)
    got = dict(zip(("h", "gx", "ggate", "gup"),
                   (h, *torch.autograd.grad(h, leaf, gh, retain_graph=True))))
    for n, v in got.items():
        oracle.close(v.reshape(vals[n].shape), vals[n], tols[n], n)
        if average and dtype != "fp32":  # (there the sums' own roundings, K of them, are the most)
            oracle.close_on_average(v, vals[n], TYPES[dtype], 1 if n == "h" else 2, n)
    again = torch.autograd.grad(h, leaf, gh)
    assert all(torch.equal(a, got[n]) for a, n in zip(again, ("gx", "ggate", "gup")))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 31, 33, 48, 64, 65, 127, 130])
def test_rows(dtype, M):
    check(M, 72, 40, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K", [1, 3, 4, 7, 8, 9, 31, 32, 63, 64, 65, 96, 127, 128, 136, 200, 260, 521])
def test_widths(dtype, K):
    check(5, K, 33, dtype)
    check(70, K, 33, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("F", [1, 2, 5, 8, 15, 16, 31, 32, 63, 64, 65, 100, 128, 129, 257])
def test_hidden_sizes(dtype, F):
    check(6, 40, F, dtype)
    check(66, 40, F, dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kind", KINDS)
def test_activations(dtype, kind):
    check(3, 64, 50, dtype, kind)
    check(80, 64, 50, dtype, kind, seed=1)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_sums_shared_by_workgroups(dtype):
    """Few tiles of x's gradient and many hidden columns; long contractions."""
    check(70, 130, 3001, dtype, average=True)
    check(9, 2000, 500, dtype)
    check(1500, 48, 72, dtype, average=True)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_largest_tiles_forward(dtype):
    check(4000, 72, 1700, dtype, average=True)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_largest_tiles_of_the_input_gradient(dtype):
    check(12200, 1030, 40, dtype, "relu" if dtype == "bf16" else "gelu")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_largest_tiles_of_the_weight_gradient(dtype):
    check(70, 2040, 3000, dtype, average=True)


def test_middle_tiles_fp32():
    check(2000, 130, 1100, "fp32")
    check(140, 1100, 1100, "fp32")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M", [20, 96])
def test_layouts(dtype, M):
    K, F = 64, 48

    def padded(by, first):
        return lambda t: torch.nn.functional.pad(t, (first, by - first)).to(DEV)[:, first:first + t.shape[1]]

    check(M, K, F, dtype, layout=padded(16, 8))    # rows on 16 bytes
    check(M, K, F, dtype, layout=padded(16, 3))    # and on none
    check(M, K, F, dtype, layout=padded(5, 0))
    check(M, K, F, dtype, layout=lambda t: t.t().contiguous().to(DEV).t())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_halves_of_one_matrix_and_more_dimensions(dtype):
    x, gate, up, gh = inputs(24, 64, 40, dtype)
    vals, tols = oracle.gated(x, gate, up, "silu", gh)
    both = torch.cat((gate, up)).to(DEV).requires_grad_()
    xd = x.view(2, 3, 4, 64).to(DEV).requires_grad_()
    h = gated_linear(xd, both[:40], both[40:])
    assert h.shape == (2, 3, 4, 40) and h.is_contiguous()
    gx, gb = torch.autograd.grad(h, [xd, both], gh.view(h.shape).to(DEV))
    oracle.close(h.view(24, 40), vals["h"], tols["h"], "h")
    oracle.close(gx.view(24, 64), vals["gx"], tols["gx"], "gx")
    oracle.close(gb, torch.cat((vals["ggate"], vals["gup"])), torch.cat((tols["ggate"], tols["gup"])), "both")
    one = gated_linear(xd[0, 0, 0].detach(), both[:40], both[40:])
    oracle.close(one[None], vals["h"][:1], tols["h"][:1], "one row")
    # the same matrix on both sides: its gradients add up
    w = gate.to(DEV).requires_grad_()
    h = gated_linear(xd, w, w)
    vals, tols = oracle.gated(x, gate, gate, "silu", gh)
    (gw,) = torch.autograd.grad(h, w, gh.view(h.shape).to(DEV))
    oracle.close(gw, vals["ggate"] + vals["gup"],
                 tols["ggate"] + tols["gup"] + oracle.half_ulp(gate.dtype) * (vals["ggate"] + vals["gup"]).abs(),
                 "shared")


@pytest.mark.parametrize("up", [2.0 ** -20, 2.0 ** -10, 16.0])
def test_gradients_in_fp16_hold_their_bits(up):
    """dg and du of every size: the whole's error is that of two roundings.  (The
    results are brought back into fp16's range by the weights.)"""
    M, K, F = 200, 64, 160
    x, gate, upw, gh = inputs(M, K, F, "fp16", up=1.0)
    gh = (gh.double() * up).half()
    vals, _ = oracle.gated(x, gate, upw, "silu", gh)
    leaf = [v.to(DEV).requires_grad_() for v in (x, gate, upw)]
    h = gated_linear(*leaf)
    got = torch.autograd.grad(h, leaf, gh.to(DEV))
    tiny = oracle.tiny(torch.float16)
    for v, n in zip(got, ("gx", "ggate", "gup")):
        err = (v.double().cpu() - vals[n]).norm()
        rounded = (vals[n].half().double() - vals[n]).norm()  # the result's own, subnormal ones included
        most = rounded + 1.05 * oracle.half_ulp(torch.float16) / 3 ** 0.5 * vals[n].norm()
        assert float(err) <= float(most), (n, float(err), float(most), tiny)


def test_gradients_in_fp16_of_large_factors():
    """Hidden values far beyond fp16's range, gradients within it."""
    x, gate, upw, gh = inputs(60, 64, 96, "fp16", up=2.0 ** -14)
    x, upw = (x.double() * 64).half(), (upw.double() * 4096).half()
    gate = (gate.double() / 64).half()
    vals, tols = oracle.gated(x, gate, upw, "gelu", gh)
    leaf = [v.to(DEV).requires_grad_() for v in (x, gate, upw)]
    h = gated_linear(*leaf, activation="gelu")
    got = torch.autograd.grad(h, leaf, gh.to(DEV))
    for v, n in zip(got, ("gx", "ggate", "gup")):
        want = vals[n]
        fits = want.abs() < 60000
        assert fits.float().mean() > 0.9
        oracle.close(torch.where(fits, v.double().cpu(), 0.0), torch.where(fits, want, 0.0), tols[n], n)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M", [40, 100])
def test_no_numbers_stay_where_they_are(dtype, M):
    """A NaN or infinity in a row of x, a weight's row or an upstream value reaches what
    the formulas say and nothing else, the neighbours of ragged tiles included."""
    K, F = 67, 45
    x, gate, up, gh = inputs(M, K, F, dtype)
    clean = [v.clone() for v in (x, gate, up, gh)]
    x[M - 1, K - 1] = float("nan")
    gate[F - 1, 0] = float("inf")
    leaf = [v.to(DEV).requires_grad_() for v in (x, gate, up)]
    h = gated_linear(*leaf)
    vals, tols = oracle.gated(*clean[:3], "silu", gh)
    assert h[M - 1].isnan().all()
    oracle.close(h[:M - 1, :F - 1], vals["h"][:M - 1, :F - 1], tols["h"][:M - 1, :F - 1], "h")
    x, gate, up, _ = clean
    gh = gh.clone()
    gh[0, 0] = float("nan")
    leaf = [v.to(DEV).requires_grad_() for v in (x, gate, up)]
    gx, gg, gu = torch.autograd.grad(gated_linear(*leaf), leaf, gh.to(DEV))
    assert gx[0].isnan().all() and gg[0].isnan().all() and gu[0].isnan().all()
    oracle.close(gx[1:], vals["gx"][1:], tols["gx"][1:], "gx")
    oracle.close(gg[1:], vals["ggate"][1:], tols["ggate"][1:], "ggate")
    oracle.close(gu[1:], vals["gup"][1:], tols["gup"][1:], "gup")


def test_empty():
    for M, K, F in ((0, 8, 8), (4, 0, 8), (4, 8, 0)):
        leaf = [torch.ones(s, device=DEV, requires_grad=True) for s in ((M, K), (F, K), (F, K))]
        h = gated_linear(*leaf)
        assert h.shape == (M, F) and not h.any()
        for g, t in zip(torch.autograd.grad(h.sum(), leaf), leaf):
            assert g.shape == t.shape and not g.any()


def test_only_what_is_asked_for():
    x, gate, up, gh = inputs(33, 24, 20, "fp32")
    vals, tols = oracle.gated(x, gate, up, "silu", gh)
    for want in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaf = [v.to(DEV).requires_grad_(i in want) for i, v in enumerate((x, gate, up))]
        gated_linear(*leaf).backward(gh.to(DEV))
        for i, n in enumerate(("gx", "ggate", "gup")):
            assert (leaf[i].grad is not None) == (i in want)
            if i in want:
                oracle.close(leaf[i].grad, vals[n], tols[n], n)

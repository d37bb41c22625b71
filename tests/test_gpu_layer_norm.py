"""layer_norm on the GPU against its formulas in 64 bits."""
from __future__ import annotations

import pytest
import torch

import block_oracle as oracle
from neural_shift_cuda import layer_norm

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda:0"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def inputs(M, n, dtype, residual=True, affine=True, seed=0, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    dt = TYPES[dtype]

    def normal(*shape, plus=0.0):
        return (torch.randn(*shape, generator=g) + plus).to(dt)

    return {"x": normal(M, n, plus=mean), "residual": normal(M, n) if residual else None,
            "weight": normal(n) if affine else None, "bias": normal(n) if affine else None,
            "gy": normal(M, n), "gs": normal(M, n) if residual else None}


def check(t, eps=1e-5, layout=lambda t: t.to(DEV), shape=None):
    """A training pass, and a forward alone, of host tensors t."""
    names = [n for n in ("x", "residual", "weight", "bias") if t[n] is not None]
    leaf = {}
    for n in names:
        v = t[n].to(DEV) if t[n].dim() == 1 else layout(t[n])
        leaf[n] = v.detach().requires_grad_()
    call = dict(weight=leaf.get("weight"), bias=leaf.get("bias"), residual=leaf.get("residual"), eps=eps)
    out = layer_norm(leaf["x"], **call)
    out = out if t["residual"] is not None else (out,)
    ups = [layout(t[n]) for n in ("gy", "gs") if t[n] is not None]
    grads = dict(zip(names, torch.autograd.grad(out, list(leaf.values()), ups)))
    vals, tols = oracle.layer_norm(t["x"], t["weight"], t["bias"], t["residual"], eps, t["gy"], t["gs"])
    flat = (lambda v: v.reshape(-1, v.shape[-1]))
    oracle.close(flat(out[0]), vals["y"], tols["y"], "y")
    if t["residual"] is not None:
        assert torch.equal(flat(out[1]).double().cpu(), vals["s"])
        assert torch.equal(grads["x"], grads["residual"])
    oracle.close(flat(grads["x"]), vals["gx"], tols["gx"], "gx")
    if t["weight"] is not None:
        oracle.close(grads["weight"], vals["gw"], tols["gw"], "gw")
        oracle.close(grads["bias"], vals["gb"], tols["gb"], "gb")
    with torch.no_grad():
        again = layer_norm(leaf["x"], **call)
        again = again if t["residual"] is not None else (again,)
        assert all(torch.equal(a, b.detach()) for a, b in zip(again, out))
    return out, grads


# around the widths where more lanes, more parts of a lane or other kernels take a row:
# 8 lanes to 64 lanes of 16 bytes, 2 and 4 parts, workgroups, rows read again
WIDTHS = [1, 2, 3, 7, 8, 9, 33, 64, 65, 128, 131, 256, 257, 511, 512, 513, 1000, 1024, 1029, 2048,
          2049, 4096, 4099, 8192, 8200, 16384, 16385, 20000]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", WIDTHS)
def test_widths(dtype, n):
    check(inputs(5, n, dtype, residual=n % 2 == 0))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("M", [1, 2, 31, 33, 600, 2101])
@pytest.mark.parametrize("n", [24, 136, 700, 1500])
def test_rows(dtype, M, n):
    check(inputs(M, n, dtype, residual=M % 2 == 0))


@pytest.mark.parametrize("n", [9000, 17000])
def test_many_wide_rows(n):
    check(inputs(700, n, "bf16"))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_without_weights(dtype):
    check(inputs(9, 200, dtype, affine=False))
    t = inputs(9, 200, dtype)
    t["bias"] = None
    leaf = [t["x"].to(DEV).requires_grad_(), t["weight"].to(DEV).requires_grad_()]
    y = layer_norm(leaf[0], leaf[1])
    got = torch.autograd.grad(y, leaf, t["gy"].to(DEV))
    vals, tols = oracle.layer_norm(t["x"], t["weight"], None, None, 1e-5, t["gy"])
    for a, n in zip((y, *got), ("y", "gx", "gw")):
        oracle.close(a, vals[n], tols[n], n)
    bias = inputs(9, 200, dtype)["bias"]
    y = layer_norm(t["x"].to(DEV), None, bias.to(DEV))
    vals, tols = oracle.layer_norm(t["x"], None, bias, None, 1e-5)
    oracle.close(y, vals["y"], tols["y"], "bias alone")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [64, 77, 2050])
def test_layouts(dtype, n):
    t = inputs(12, n, dtype)
    check(t, layout=lambda v: torch.nn.functional.pad(v, (3, 2)).to(DEV)[:, 3:3 + n])
    check(t, layout=lambda v: v.t().contiguous().to(DEV).t())
    check(t, layout=lambda v: v.view(3, 4, n).to(DEV))
    check(t, layout=lambda v: v.view(3, 4, n).transpose(0, 1).contiguous().to(DEV).transpose(0, 1))
    check(t, layout=lambda v: v.view(3, 4, 1, n).transpose(1, 2).to(DEV))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_mean_far_from_the_deviations(dtype):
    check(inputs(6, 500, dtype, residual=False, mean=200.0))


def test_rows_of_one_value():
    for n in (8, 300, 5000):
        x = torch.full((4, n), 3.25, device=DEV, requires_grad=True)
        y = layer_norm(x)
        assert not y.any()
        (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
        # 1 less the mean of ones, which 1 / n, a product and a sum round: three steps of
        # 2^-24, over sqrt(eps)
        assert float(g.abs().max()) <= 3 * oracle.F32 / 1e-5 ** 0.5


def test_no_numbers_stay_in_their_rows():
    for n in (40, 900, 3000, 9000, 17000):
        t = inputs(6, n, "fp32")
        t["x"][1, n // 2] = float("nan")
        t["x"][3, 0] = float("inf")
        leaf = [t[k].to(DEV).requires_grad_() for k in ("x", "residual", "weight", "bias")]
        y, s = layer_norm(leaf[0], leaf[2], leaf[3], residual=leaf[1])
        grads = torch.autograd.grad([y, s], leaf, [t["gy"].to(DEV), t["gs"].to(DEV)])
        ok = [0, 2, 4, 5]
        vals, tols = oracle.layer_norm(t["x"][ok], t["weight"], t["bias"], t["residual"][ok], 1e-5,
                                       t["gy"][ok], t["gs"][ok])
        oracle.close(y[ok], vals["y"], tols["y"], "y")
        oracle.close(grads[0][ok], vals["gx"], tols["gx"], "gx")
        assert y[1].isnan().all() and y[3].isnan().all()
        oracle.close(grads[3], t["gy"].double().sum(0), 20 * oracle.F32 * t["gy"].abs().sum(0), "gb")


def test_empty():
    w = torch.ones(16, device=DEV, requires_grad=True)
    x = torch.empty(2, 0, 16, device=DEV, requires_grad=True)
    y, s = layer_norm(x, w, residual=x.detach())
    assert y.shape == s.shape == (2, 0, 16)
    gx, gw = torch.autograd.grad(y.sum(), [x, w])
    assert gx.shape == x.shape and not gw.any()
    x = torch.empty(3, 0, device=DEV, requires_grad=True)
    assert torch.autograd.grad(layer_norm(x).sum(), x)[0].shape == (3, 0)


def test_only_what_is_asked_for():
    t = inputs(7, 96, "fp32")
    vals, tols = oracle.layer_norm(t["x"], t["weight"], t["bias"], t["residual"], 1e-5, t["gy"], t["gs"])
    names = {"x": "gx", "residual": "gx", "weight": "gw", "bias": "gb"}
    for want in (["x"], ["residual"], ["weight"], ["bias"], ["residual", "bias"], ["x", "weight"]):
        leaf = {n: t[n].to(DEV).requires_grad_(n in want) for n in names}
        y, s = layer_norm(leaf["x"], leaf["weight"], leaf["bias"], residual=leaf["residual"])
        torch.autograd.backward([y, s] if "x" in want or "residual" in want else [y],
                                [t["gy"].to(DEV), t["gs"].to(DEV)][:2 if s.requires_grad and (
                                    "x" in want or "residual" in want) else 1])
        for n in names:
            assert (leaf[n].grad is not None) == (n in want), (want, n)
            if n in want:
                oracle.close(leaf[n].grad, vals[names[n]], tols[names[n]], n)


def test_one_gradient_of_the_stream_alone():
    t = inputs(7, 96, "fp32")
    leaf = {n: t[n].to(DEV).requires_grad_() for n in ("x", "residual", "weight")}
    _, s = layer_norm(leaf["x"], leaf["weight"], residual=leaf["residual"])
    gx, gr, gw = torch.autograd.grad(s, list(leaf.values()), t["gs"].to(DEV))
    assert torch.equal(gx.cpu(), t["gs"]) and torch.equal(gr.cpu(), t["gs"]) and not gw.any()

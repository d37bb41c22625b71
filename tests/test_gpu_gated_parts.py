"""The gated projections in fp32 where they are taken apart into sums of three bf16
numbers: the values that such sums might lose."""
from __future__ import annotations

import ctypes

import pytest
import torch

import block_oracle as oracle
from neural_shift_cuda import gated_linear
from neural_shift_cuda_amd import _C

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda:0"
M, K, F = 2000, 132, 1100  # rows on whole 16 bytes: nothing is copied but for the parts


def inputs(seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(M, K, generator=g), torch.randn(F, K, generator=g) * K ** -0.5,
            torch.randn(F, K, generator=g) * K ** -0.5, torch.randn(M, F, generator=g)]


def run(x, gate, up, gh, kind="silu"):
    leaf = [t.to(DEV).requires_grad_() for t in (x, gate, up)]
    h = gated_linear(*leaf, activation=kind)
    return dict(zip(("h", "gx", "ggate", "gup"), (h, *torch.autograd.grad(h, leaf, gh.to(DEV)))))


def check(x, gate, up, gh, kind="silu", rows=slice(None), names=("h", "gx", "ggate", "gup")):
    vals, tols = oracle.gated(x, gate, up, kind, gh)
    got = run(x, gate, up, gh, kind)
    for n in names:
        pick = rows if n in ("h", "gx") else slice(None)
        oracle.close(got[n][pick], vals[n][pick], tols[n][pick], n)
    return got


@pytest.mark.parametrize("backward", [0, 1])
def test_these_sizes_are_taken_apart(backward):
    """The workspace holds the parts: 6 bytes an element of x and the weights."""
    a = _C._GatedLinearArgs()
    one = torch.empty(64, device=DEV).data_ptr()
    for n in ("x", "gate_weight", "up_weight", "h", "kept", "grad_h", "grad_x", "grad_gate", "grad_up"):
        setattr(a, n, one)
    a.rows, a.K, a.F, a.x_stride, a.gate_stride, a.up_stride, a.gh_stride = M, K, F, K, K, K, F
    a.dtype, a.activation = 3, 1
    got = _C._lib.nsh_gated_linear_workspace_bytes(ctypes.byref(a), backward)
    assert got >= 6 * (M + 2 * F) * K


@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
def test_values(kind):
    check(*inputs(), kind)


def test_whole_numbers_are_exact():
    """Products of small whole numbers: not a bit of the sums is lost."""
    g = torch.Generator().manual_seed(1)
    x, gate, up, gh = (torch.randint(-8, 9, s, generator=g).float() for s in ((M, K), (F, K), (F, K), (M, F)))
    vals, _ = oracle.gated(x, gate, up, "relu", gh)
    assert torch.equal(run(x, gate, up, gh, "relu")["h"].cpu().double(), vals["h"])


def test_numbers_of_24_bits_times_a_power_of_two():
    """One weight a row: h has x's own bits, of which 3 x 8 are kept."""
    x, gate, up, gh = inputs(2)
    gate, up = torch.zeros_like(gate), torch.zeros_like(up)
    gate[:, 0], up[:, 1] = 4.0, 0.5
    x[:, 0], x[:, 1] = 1.0, torch.rand(M, generator=torch.Generator().manual_seed(3)) + 1.0
    assert torch.equal(run(x, gate, up, gh, "relu")["h"].cpu(), (x[:, 1:2] * 2).expand(M, F))


def test_rows_of_different_sizes():
    x, gate, up, gh = inputs(4)
    size = 2.0 ** torch.randint(-24, 4, (M, 1), generator=torch.Generator().manual_seed(5)).float()
    check(x * size, gate, up, gh)
    check(x, gate, up, gh * size)


def test_large_and_small_sides():
    """x near fp32's end, beyond bf16's, times weights as small."""
    x, gate, up, gh = inputs(6)
    big = torch.finfo(torch.float32).max
    x = (x * 2.0 ** 100).clamp(-big, big)
    x[:, 0] = big
    gate, up = gate * 2.0 ** -100, up * 2.0 ** -100
    gate[:, 0], up[:, 0] = 2.0 ** -128, 2.0 ** -127
    check(x, gate, up, gh, names=("h",))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_is_no_number_stays_in_its_place(bad):
    x, gate, up, gh = inputs(7)
    clean = oracle.gated(x, gate, up, "silu", gh)
    x2 = x.clone()
    x2[M - 1, 3] = bad
    got = run(x2, gate, up, gh)
    assert not got["h"][M - 1].isfinite().any()
    oracle.close(got["h"][:-1], clean[0]["h"][:-1], clean[1]["h"][:-1], "h")
    oracle.close(got["gx"][:-1], clean[0]["gx"][:-1], clean[1]["gx"][:-1], "gx")
    assert not got["ggate"][:, 3].isfinite().any()
    g2 = gate.clone()
    g2[F - 1, K - 1] = bad
    h = run(x, g2, up, gh)["h"]
    oracle.close(h[:, :-1], clean[0]["h"][:, :-1], clean[1]["h"][:, :-1], "h")
    assert not (h[:, -1].isfinite() & (h[:, -1] != 0)).any()  # silu(-inf) is 0 or no number
    gh2 = gh.clone()
    gh2[0, 5] = bad
    got = run(x, gate, up, gh2)
    assert not got["gx"][0].isfinite().any()
    oracle.close(got["gx"][1:], clean[0]["gx"][1:], clean[1]["gx"][1:], "gx")
    rest = [i for i in range(F) if i != 5]
    for n in ("ggate", "gup"):
        assert not got[n][5].isfinite().any()
        oracle.close(got[n][rest], clean[0][n][rest], clean[1][n][rest], n)


def test_an_infinity_is_one():
    """An infinity times numbers is the infinity that fp32 would have."""
    x, gate, up, gh = inputs(8)
    x[0, 0] = float("inf")
    want = (x.double() @ gate.double().t()).relu() * (x.double() @ up.double().t())
    got = run(x, gate, up, gh, "relu")["h"][0].cpu().double()
    ok = want[0].isnan() == got.isnan()
    assert ok.all() and torch.equal(got[got.isinf()], want[0][got.isinf()])

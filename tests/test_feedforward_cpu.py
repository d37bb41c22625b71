"""layer_norm and gated_linear: their CPU forms against torch's and against
differences, the oracle's formulas against the CPU forms, refusals, and the C
entries' checks."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import block_oracle as oracle
from neural_shift_cuda import gated_linear, gated_linear_reference, layer_norm, layer_norm_reference

KINDS = ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]


def rand(*shape, seed=0, dtype=torch.float64):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape)), dtype=dtype)


def test_layer_norm_is_torchs():
    x, w, b = rand(3, 4, 10), rand(10), rand(10, seed=1)
    torch.testing.assert_close(layer_norm(x, w, b, eps=1e-3),
                               torch.nn.functional.layer_norm(x, (10,), w, b, 1e-3))
    y, s = layer_norm(x, w, residual=x * 2)
    torch.testing.assert_close(s, 3 * x)
    torch.testing.assert_close(y, torch.nn.functional.layer_norm(3 * x, (10,), w))
    x = x.bfloat16()
    y, s = layer_norm(x, residual=x)
    assert y.dtype == s.dtype == torch.bfloat16 and torch.equal(s, x + x)
    assert torch.equal(y, layer_norm(s))
    assert layer_norm(torch.empty(3, 0)).shape == (3, 0)


def test_layer_norm_gradients_against_differences():
    x, r, w, b = (rand(3, 6, seed=i) if i < 2 else rand(6, seed=i) for i in range(4))
    leaves = [t.requires_grad_() for t in (x, r, w, b)]
    assert torch.autograd.gradcheck(lambda x, r, w, b: layer_norm_reference(x, w, b, residual=r), leaves)


@pytest.mark.parametrize("kind", KINDS)
def test_gated_gradients_against_differences(kind):
    leaves = [t.requires_grad_() for t in (rand(3, 5), rand(4, 5), rand(4, 5, seed=1))]
    assert torch.autograd.gradcheck(lambda *t: gated_linear_reference(*t, activation=kind), leaves)


@pytest.mark.parametrize("kind", KINDS)
def test_the_oracles_formulas(kind):
    x, gate, up, gh = rand(7, 5), rand(6, 5), rand(6, 5, seed=1), rand(7, 6)
    vals, tols = oracle.gated(x, gate, up, kind, gh)
    leaves = [t.clone().requires_grad_() for t in (x, gate, up)]
    h = gated_linear(*leaves, activation=kind)
    torch.testing.assert_close(h.detach(), vals["h"])
    for g, n in zip(torch.autograd.grad(h, leaves, gh), ("gx", "ggate", "gup")):
        torch.testing.assert_close(g, vals[n])
    # what the tolerance is for: fp32 inside it, and not by far
    single, t32 = oracle.gated(*(t.float() for t in (x, gate, up)), kind, gh.float())
    leaves = [t.float().requires_grad_() for t in (x, gate, up)]
    h = gated_linear(*leaves, activation=kind)
    oracle.close(h, single["h"], t32["h"], "h")
    assert float((t32["h"] / single["h"].abs().mean()).max()) < 1e-3


def test_the_oracles_layer_norm():
    x, r, w, b, gy, gs = rand(5, 9), rand(5, 9, seed=1), rand(9), rand(9, seed=1), rand(5, 9, seed=2), rand(5, 9, seed=3)
    x, r = x.float().double(), r.float().double()  # (the oracle adds the two in fp32)
    s = (x.float() + r.float()).double()
    leaves = [t.clone().requires_grad_() for t in (s, w, b)]
    y = layer_norm(*leaves)
    vals, _ = oracle.layer_norm(x, w, b, r, 1e-5, gy, gs)
    torch.testing.assert_close(y.detach(), vals["y"])
    gx, gw, gb = torch.autograd.grad(y, leaves, gy)
    for a, n in ((gx + gs, "gx"), (gw, "gw"), (gb, "gb")):
        torch.testing.assert_close(a, vals[n])


def refused(error, match, f, *a, **k):
    with pytest.raises(error, match=match):
        f(*a, **k)


def test_layer_norm_refusals():
    x, w = rand(3, 8), rand(8)
    f = layer_norm
    refused(ValueError, "width", f, torch.tensor(1.0))
    refused(TypeError, "floating", f, x.long())
    refused(ValueError, "weight must be", f, x, w[:4])
    refused(ValueError, "bias must be", f, x, w, rand(1, 8))
    refused(ValueError, "weight must have dtype", f, x, w.float())
    refused(ValueError, "residual must be", f, x, residual=x[:2])
    refused(ValueError, "residual must have dtype", f, x, residual=x.float())
    for bad in (-1.0, math.nan, math.inf):
        refused(ValueError, "eps", f, x, eps=bad)


def test_gated_refusals():
    x, w = rand(3, 8), rand(5, 8)
    f = gated_linear
    refused(ValueError, "width", f, torch.tensor(1.0), w, w)
    refused(TypeError, "floating", f, x.long(), w, w)
    refused(ValueError, "hidden", f, x, w[:, :4], w[:, :4])
    refused(ValueError, "hidden", f, x, w, w[:4])
    refused(ValueError, "hidden", f, x, w[0], w[0])
    refused(ValueError, "dtype", f, x, w.float(), w)
    refused(ValueError, "dtype", f, x, w, w.float())
    refused(ValueError, "activation", f, x, w, w, activation="tanh")
    refused(ValueError, "activation", f, x, w, w, activation=None)


# the C entries check on the host before any device work
def native():
    from neural_shift_cuda_amd import _C
    return _C


@pytest.mark.parametrize("over,match", [
    ({"dtype": 4}, "dtype"), ({"dtype": 0}, "dtype"), ({"rows": 0}, "empty"), ({"n": 0}, "empty"),
    ({"n": 1 << 31}, "2\\^30"), ({"rows": 1 << 41}, "2\\^40"), ({"eps": -1.0}, "eps"),
    ({"eps": math.nan}, "eps"), ({"x": None}, "null"), ({"y": None}, "null"), ({"s": 16}, "null"),
    ({"residual": 16}, "null")])
def test_layer_norm_entry_checks(over, match):
    C = native()
    a = dict(x=16, y=16, rows=2, n=8, x_stride=8, eps=1e-5, dtype=3)
    with pytest.raises(RuntimeError, match=match):
        C._call("nsh_layer_norm_forward", ctypes.byref(C._LayerNormArgs(**{**a, **over})), None)


def test_layer_norm_backward_entry_checks():
    C = native()
    a = dict(x=16, rows=2, n=8, x_stride=8, eps=1e-5, dtype=3, grad_y=16, gy_stride=8, stats=16)
    for over, match in (({}, "null"), ({"grad_x": 16, "stats": None}, "null"),
                        ({"grad_weight": 16}, "workspace"),
                        ({"grad_bias": 16, "workspace": 16, "workspace_bytes": 8}, "workspace"),
                        ({"grad_bias": 16, "workspace": 17, "workspace_bytes": 1 << 20}, "misaligned")):
        with pytest.raises(RuntimeError, match=match):
            C._call("nsh_layer_norm_backward", ctypes.byref(C._LayerNormArgs(**{**a, **over})), None)


@pytest.mark.parametrize("over,match", [
    ({"dtype": 4}, "dtype"), ({"rows": 0}, "empty"), ({"K": 0}, "empty"), ({"F": 0}, "empty"),
    ({"K": (1 << 20) + 1}, "2\\^20"), ({"F": (1 << 20) + 1}, "2\\^20"), ({"rows": 1 << 31}, "2\\^30"),
    ({"activation": 0}, "activation"), ({"activation": 6}, "activation"), ({"x": None}, "null"),
    ({"up_weight": None}, "null"), ({"h": None}, "null"), ({"kept": 8}, "misaligned"),
    ({"x": 8}, "workspace"), ({"K": 7}, "workspace"), ({"gate_stride": 12}, "workspace"),
    ({"x_stride": 0}, "workspace"), ({"x_stride": 1 << 30}, "workspace"),
    ({"K": 7, "workspace": 24, "workspace_bytes": 1 << 20}, "misaligned")])
def test_gated_entry_checks(over, match):
    C = native()
    a = dict(x=16, gate_weight=16, up_weight=16, rows=2, K=8, F=4, x_stride=8, gate_stride=8,
             up_stride=8, dtype=2, activation=1, h=16)
    with pytest.raises(RuntimeError, match=match):
        C._call("nsh_gated_linear_forward", ctypes.byref(C._GatedLinearArgs(**{**a, **over})), None)


def test_gated_backward_entry_checks():
    C = native()
    a = dict(x=16, gate_weight=16, up_weight=16, rows=2, K=8, F=4, x_stride=8, gate_stride=8,
             up_stride=8, dtype=2, activation=1, kept=16, grad_h=16, gh_stride=4)
    for over, match in (({}, "null"), ({"grad_x": 16, "kept": None}, "null"),
                        ({"grad_x": 16, "grad_h": None}, "null"), ({"grad_x": 16}, "workspace")):
        with pytest.raises(RuntimeError, match=match):
            C._call("nsh_gated_linear_backward", ctypes.byref(C._GatedLinearArgs(**{**a, **over})), None)
    for name in ("nsh_layer_norm_forward", "nsh_layer_norm_backward", "nsh_gated_linear_forward",
                 "nsh_gated_linear_backward"):
        with pytest.raises(RuntimeError, match="null"):
            C._call(name, None, None)


def test_workspaces_grow_with_what_is_copied():
    C = native()
    a = dict(x=16, gate_weight=16, up_weight=16, rows=300, K=64, F=40, x_stride=64, gate_stride=64,
             up_stride=64, dtype=2, activation=1)

    def size(backward=0, **over):
        return C._lib.nsh_gated_linear_workspace_bytes(ctypes.byref(C._GatedLinearArgs(**{**a, **over})), backward)

    assert size() == 0
    assert size(x=18) >= 300 * 64 * 2
    assert size(gate_weight=18, up_weight=20) >= 2 * 40 * 64 * 2
    assert size(K=63) >= (300 + 2 * 40) * 64 * 2
    assert size(1) >= 300 * 2 * 64 * 2
    assert size(rows=0) == -1
    assert C._lib.nsh_gated_linear_kept_bytes(ctypes.byref(C._GatedLinearArgs(**a))) >= 300 * 2 * 40 * 2
    assert C._lib.nsh_layer_norm_workspace_bytes(None) == -1


def test_struct_sizes_match_the_header(tmp_path):
    import os
    import shutil
    import subprocess
    cc = shutil.which("gcc")
    if not cc:
        pytest.skip("no C compiler")
    C = native()
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "neural_shift_hip.h"\n'
                   'int main(){printf("%zu %zu %zu %zu", sizeof(nsh_layer_norm_args), '
                   'offsetof(nsh_layer_norm_args, grad_y), sizeof(nsh_gated_linear_args), '
                   'offsetof(nsh_gated_linear_args, kept));}')
    exe = tmp_path / "s"
    subprocess.run([cc, "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    L, G = C._LayerNormArgs, C._GatedLinearArgs
    assert got == [ctypes.sizeof(L), L.grad_y.offset, ctypes.sizeof(G), G.kept.offset]

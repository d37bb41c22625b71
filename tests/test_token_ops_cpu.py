"""The token operators on the CPU: the reference implementations against the
formulas in 64 bits, their gradients against differences, and what the
operators refuse."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import token_oracle as oracle
from neural_shift_cuda import (biased_attention, qk_norm_rotary, relative_buckets,
                               relative_position_bias, rotary_table)

F64 = torch.float64


def rand(*shape, seed=0, dtype=F64):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=dtype)


CASES = {
    "plain": {},
    "causal": {"causal": True},
    "cap": {"cap": 3.0, "scale": 0.4},
    "prefix": {"causal": True, "prefix": torch.tensor([3, 9])},
    "lengths": {"causal": True, "lengths": torch.tensor([13, 0])},
    "documents": {"documents": torch.tensor([[0] * 4 + [1] * 5 + [-1] * 4, [2] * 13])},
    "slopes": {"slopes": torch.tensor([0.1, 0.2, 0.0, 1.0], dtype=F64)},
    "buckets": {"bias_table": rand(8, 4, seed=9), "buckets": relative_buckets(8, 6)},
}


@pytest.mark.parametrize("name", list(CASES))
def test_reference_attention(name):
    rules = CASES[name]
    q, go = rand(2, 4, 7, 6), rand(2, 4, 7, 6, seed=3)
    k, v = rand(2, 2, 13, 6, seed=1), rand(2, 2, 13, 6, seed=2)
    vals, _ = oracle.attention(q, k, v, go=go, **rules)
    leaves = {"gq": q, "gk": k, "gv": v}
    if "bias_table" in rules:
        leaves["gtable"] = rules["bias_table"]
    leaves = {n: t.clone().requires_grad_() for n, t in leaves.items()}
    rules = {**rules, **({"bias_table": leaves["gtable"]} if "gtable" in leaves else {})}
    out, degree = biased_attention(leaves["gq"], leaves["gk"], leaves["gv"],
                                   return_log_degree=True, **rules)
    tol = torch.tensor(1e-12)
    oracle.close(out, vals["out"], tol, "out")
    oracle.close(degree, vals["degree"], tol, "degree")
    for n, g in zip(leaves, torch.autograd.grad(out, list(leaves.values()), go)):
        oracle.close(g, vals[n], tol, n)


def test_unseen_keys_are_not_used():
    q, k, v = rand(1, 1, 3, 4), rand(1, 1, 6, 4, seed=1), rand(1, 1, 6, 4, seed=2)
    want = biased_attention(q, k[:, :, :4], v[:, :, :4])
    k[:, :, 4:], v[:, :, 4:] = math.nan, math.inf
    got = biased_attention(q, k, v, lengths=torch.tensor([4]))
    oracle.close(got, want, torch.tensor(1e-13), "out")


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(8, 8), (7, 4), (6, 0)])
def test_reference_norm(interleaved, D, rot):
    x, g, w = rand(2, 3, 4, D), rand(2, 3, 4, D, seed=1), rand(D, seed=2)
    cos, sin = rotary_table(9, rot)
    at = torch.tensor([[0, 8, 3, 9], [1, -1, 2, 5]])
    leaf, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
    out = qk_norm_rotary(leaf, x[:, :1], wl, None, cos, sin, at, interleaved=interleaved)[0]
    gx, gw = torch.autograd.grad(out, (leaf, wl), g)
    vals, _ = oracle.norm_rotary(x, w, cos, sin, at, 1e-6, interleaved, g)
    for got, n in ((out, "out"), (gx, "gx"), (gw, "gw")):
        if rot and n != "out":
            continue  # NaN spreads through the gradient's sums; checked below
        oracle.close(got, vals[n], torch.tensor(1e-12), n)
    at = at.clamp(0, 8)
    out = qk_norm_rotary(leaf, x[:, :1], wl, None, cos, sin, at, interleaved=interleaved)[0]
    vals, _ = oracle.norm_rotary(x, w, cos, sin, at, 1e-6, interleaved, g)
    for got, n in zip((out, *torch.autograd.grad(out, (leaf, wl), g)), ("out", "gx", "gw")):
        oracle.close(got, vals[n], torch.tensor(1e-12), n)


def test_reference_bias():
    table, buckets = rand(8, 3), relative_buckets(8, 5)
    for Lq, Lk in ((4, 4), (1, 9), (7, 3)):
        leaf, go = table.clone().requires_grad_(), rand(3, Lq, Lk, seed=4)
        out = relative_position_bias(leaf, buckets, Lq, Lk)
        assert torch.equal(out.detach(), oracle.position_bias(table, buckets, Lq, Lk))
        (g,) = torch.autograd.grad(out, leaf, go)
        oracle.close(g, oracle.position_bias_grad(go, buckets, 8)[0], torch.tensor(1e-12), "grad")


def test_gradcheck():
    q, k, v = (rand(1, 2, 3, 4, seed=s).requires_grad_() for s in range(3))
    table = rand(4, 2, seed=5).requires_grad_()
    buckets = relative_buckets(4, 3)
    assert torch.autograd.gradcheck(
        lambda *t: biased_attention(*t[:3], cap=2.0, causal=True, bias_table=t[3],
                                    buckets=buckets, return_log_degree=True), (q, k, v, table))
    w = rand(4, seed=6).requires_grad_()
    cos, sin = rotary_table(3, 4)
    assert torch.autograd.gradcheck(lambda a, b, c: qk_norm_rotary(a, b, c, c, cos, sin), (q, k, w))


def test_rotary_table():
    cos, sin = rotary_table(100001, 6, base=500.0)
    for p, i in ((0, 0), (7, 1), (100000, 0), (100000, 2)):
        a = p * 500.0 ** (-2 * i / 6)
        assert abs(float(cos[p, i]) - math.cos(a)) <= 2.0 ** -24
        assert abs(float(sin[p, i]) - math.sin(a)) <= 2.0 ** -24
    grid = torch.stack(torch.meshgrid(torch.arange(3), torch.arange(5), indexing="ij"), -1)
    cos, _ = rotary_table(grid.view(-1, 2), 8)
    rows, cols = rotary_table(3, 4)[0], rotary_table(5, 4)[0]
    assert torch.equal(cos.view(3, 5, 4)[1, 4], torch.cat((rows[1], cols[4])))


def test_relative_buckets():
    b = relative_buckets(32, 128)
    rel = range(-128, 129)
    assert b.dtype == torch.int32 and [int(x) for x in b[128 - 7:129]] == [7, 6, 5, 4, 3, 2, 1, 0]
    assert [int(x) for x in b[129:129 + 7]] == [17, 18, 19, 20, 21, 22, 23]
    assert int(b[0]) == 15 and int(b[-1]) == 31
    for r, x in zip(rel, b.tolist()):
        d = abs(r)
        want = d if d < 8 else min(15, 8 + int(math.log(d / 8) / math.log(16) * 8))
        assert x == want + (16 if r > 0 else 0)
    one = relative_buckets(16, 64, bidirectional=False)
    assert not one[64:].any() and int(one[0]) == 15


def refused(error, match, f, *a, **k):
    with pytest.raises(error, match=match):
        f(*a, **k)


def test_attention_refusals():
    q, k = rand(2, 4, 3, 8), rand(2, 2, 5, 8)
    f = biased_attention
    refused(ValueError, "q must be", f, q[0], k, k)
    refused(TypeError, "floating", f, q.long(), k, k)
    refused(ValueError, "dtype", f, q, k.float(), k)
    refused(ValueError, "k and v", f, q, k, k[:, :, :4])
    refused(ValueError, "k and v", f, q, k[..., :4], k[..., :4])
    refused(ValueError, "multiple", f, q[:, :3], k, k)
    refused(ValueError, "head width", f, q[..., :0], k[..., :0], k[..., :0])
    for bad in (math.nan, math.inf, -1.0):
        refused(ValueError, "finite", f, q, k, k, cap=bad)
    refused(ValueError, "finite", f, q, k, k, scale=math.inf)
    refused(ValueError, "causal", f, q, k, k, prefix=torch.tensor([1, 1]))
    refused(ValueError, "lengths", f, q, k, k, lengths=torch.tensor([1]))
    refused(TypeError, "lengths", f, q, k, k, lengths=torch.tensor([1.0, 2.0]))
    refused(TypeError, "documents", f, q, k, k, documents=torch.zeros(2, 5, dtype=torch.bool))
    refused(ValueError, "documents", f, q, k, k, documents=torch.zeros(2, 3, dtype=torch.int32))
    refused(ValueError, "slopes", f, q, k, k, slopes=rand(2))
    refused(TypeError, "slopes", f, q, k, k, slopes=torch.ones(4, dtype=torch.int32))
    refused(ValueError, "no gradient", f, q, k, k, slopes=rand(4).requires_grad_())
    table, buckets = rand(8, 4), relative_buckets(8, 4)
    refused(ValueError, "buckets", f, q, k, k, bias_table=table)
    refused(ValueError, "bias_table", f, q, k, k, buckets=buckets)
    refused(ValueError, "buckets", f, q, k, k, bias_table=table, buckets=buckets[1:])
    refused(ValueError, "heads", f, q, k, k, bias_table=table[:, :2], buckets=buckets)
    refused(ValueError, "dtype", f, q, k, k, bias_table=table.float(), buckets=buckets)
    refused(ValueError, "reach", f, q, k, k, bias_table=table,
            buckets=torch.zeros(4099, dtype=torch.int32))


def test_norm_refusals():
    q, k, w = rand(2, 4, 3, 8), rand(2, 2, 3, 8), rand(8)
    cos, sin = rotary_table(5, 8)
    f = qk_norm_rotary
    refused(ValueError, "agree", f, q, k[:, :, :2], w, w, cos, sin)
    refused(ValueError, "q_weight", f, q, k, w[:4], w, cos, sin)
    refused(ValueError, "dtype", f, q, k, w.float(), w, cos, sin)
    refused(ValueError, "cos and sin", f, q, k, w, w, cos, sin[:, :2])
    refused(ValueError, "cos and sin", f, q[..., :6], k[..., :6], w[:6], w[:6], cos, sin)
    refused(TypeError, "float32", f, q, k, w, w, cos.half(), sin.half())
    refused(ValueError, "rows", f, q, k, w, w, cos[:2], sin[:2])
    refused(ValueError, "positions", f, q, k, w, w, cos, sin, torch.zeros(2, 4, dtype=torch.int64))
    refused(TypeError, "positions", f, q, k, w, w, cos, sin, torch.zeros(3))
    refused(ValueError, "even", rotary_table, 4, 7)
    refused(ValueError, "axes", rotary_table, torch.zeros(4, 2), 6)


def test_bias_refusals():
    table, buckets = rand(8, 4), relative_buckets(8, 4)
    f = relative_position_bias
    refused(ValueError, "negative", f, table, buckets, -1, 3)
    refused(ValueError, "table", f, table[0], buckets, 2, 3)
    refused(ValueError, "buckets", f, table, buckets[:-1], 2, 3)
    refused(TypeError, "buckets", f, table, buckets.float(), 2, 3)
    refused(TypeError, "floating", f, table.long(), buckets, 2, 3)
    refused(ValueError, "relative_buckets", relative_buckets, 2, 10)
    refused(ValueError, "relative_buckets", relative_buckets, 64, 10)
    refused(ValueError, "relative_buckets", relative_buckets, 32, 4096)


# the C entries check on the host before any device work
def native():
    from neural_shift_cuda_amd import _C
    return _C


def attention_args(**over):
    C = native()
    a = dict(q=16, k=16, v=16, out=16, B=1, Hq=2, Hk=1, Lq=4, Lk=4, D=8, q_stride=(64, 32, 8),
             k_stride=(32, 32, 8), v_stride=(32, 32, 8), out_stride=(64, 32, 8), scale=1.0, cap=0.0,
             dtype=2, causal=1)
    return C._AttentionArgs(**{**a, **over})


@pytest.mark.parametrize("over,match", [
    ({"dtype": 4}, "dtype"), ({"dtype": 0}, "dtype"), ({"B": 0}, "empty"), ({"Lk": 0}, "empty"),
    ({"Lq": 1 << 31}, "2\\^30"), ({"B": 1 << 28, "Hq": 16, "Hk": 16}, "2\\^30"), ({"Hk": 3}, "multiple"),
    ({"D": 12}, "width"), ({"D": 136}, "width"), ({"cap": -1.0}, "finite"),
    ({"cap": math.nan}, "finite"), ({"scale": math.inf}, "finite"),
    ({"prefix": 16, "causal": 0}, "prefix"), ({"bias_table": 16}, "buckets"),
    ({"bias_table": 16, "buckets": 16, "num_buckets": 4, "reach": 2049}, "reach"),
    ({"k": None}, "null"), ({"q": 8}, "16 bytes"), ({"k_stride": (32, 32, 9)}, "16 bytes")])
def test_attention_entry_checks(over, match):
    C = native()
    with pytest.raises(RuntimeError, match=match):
        C._call("nsh_attention_forward", ctypes.byref(attention_args(**over)), None)


def test_backward_entry_checks():
    C = native()
    with pytest.raises(RuntimeError, match="null"):
        C._call("nsh_attention_backward", ctypes.byref(attention_args()), None)
    a = attention_args(log_degree=16, grad_out=16, grad_q=16, grad_k=16, grad_v=16,
                       go_stride=(64, 32, 8), gq_stride=(64, 32, 8), gk_stride=(32, 32, 8),
                       gv_stride=(32, 32, 8))
    with pytest.raises(RuntimeError, match="workspace"):
        C._call("nsh_attention_backward", ctypes.byref(a), None)
    a.go_stride[2] = 9
    with pytest.raises(RuntimeError, match="16 bytes"):
        C._call("nsh_attention_backward", ctypes.byref(a), None)
    for name in ("nsh_attention_forward", "nsh_attention_backward", "nsh_norm_rotary_forward"):
        with pytest.raises(RuntimeError, match="null"):
            C._call(name, None, None)


def test_other_entry_checks():
    C = native()
    a = dict(q=16, k=16, q_out=16, k_out=16, cos=16, sin=16, B=1, Hq=1, Hk=1, L=1, D=8, half=4,
             rows=1, q_stride=(8, 8, 8), k_stride=(8, 8, 8), eps=1e-6, dtype=3)
    for over, match in (({"dtype": 4}, "dtype"), ({"D": 513}, "width"), ({"half": 5}, "width"),
                        ({"B": 0}, "empty"), ({"L": 1 << 31}, "rows"), ({"cos": None}, "cos"),
                        ({"q": None}, "null"), ({"k_out": None}, "null")):
        with pytest.raises(RuntimeError, match=match):
            C._call("nsh_norm_rotary_forward", ctypes.byref(C._NormRotaryArgs(**{**a, **over})), None)
    g = C._NormRotaryArgs(**a, grad_q_out=16, grad_k_out=16, grad_q=16, grad_k=16, grad_q_weight=16)
    with pytest.raises(RuntimeError, match="workspace"):
        C._call("nsh_norm_rotary_backward", ctypes.byref(g), None)
    for args, match in (((16, 16, 0, 1, 1, 1, 0, 3, 16, None), "empty"),
                        ((16, 16, 1, 1, 1, 1, 2049, 3, 16, None), "reach"),
                        ((16, 16, 1, 1, 1, 1, 0, 4, 16, None), "dtype"),
                        ((16, 16, 70000, 1, 1, 1, 0, 3, 16, None), "65535"),
                        ((16, None, 1, 1, 1, 1, 0, 3, 16, None), "null")):
        with pytest.raises(RuntimeError, match=match):
            C._call("nsh_position_bias_forward", *args)
    with pytest.raises(RuntimeError, match="workspace"):
        C._call("nsh_position_bias_backward", 16, 16, 1, 64, 64, 1, 4, 3, 16, 16, 8, None)


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
                   'int main(){printf("%zu %zu %zu %zu", sizeof(nsh_attention_args), '
                   'offsetof(nsh_attention_args, grad_q), sizeof(nsh_norm_rotary_args), '
                   'offsetof(nsh_norm_rotary_args, eps));}')
    exe = tmp_path / "s"
    subprocess.run([cc, "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True,
                                          check=True).stdout.split()]
    A, N = C._AttentionArgs, C._NormRotaryArgs
    assert got == [ctypes.sizeof(A), A.grad_q.offset, ctypes.sizeof(N), N.eps.offset]

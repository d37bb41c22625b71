"""Layer norm and the gated projections as a program calls them: on other streams, in
graphs, in traces, with their saved tensors elsewhere, and together."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import block_oracle as oracle
from neural_shift_cuda import gated_linear, layer_norm
from test_gpu_layer_norm import check as check_norm, inputs as norm_inputs

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]
DEV = "cuda"


def tensors(*shapes, dtype=torch.float32, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(*s, generator=g).to(DEV, dtype) for s in shapes]


def gated_leaves(M, K, F, dtype):
    x, gate, up = tensors((M, K), (F, K), (F, K), dtype=dtype)
    return [x, gate * K ** -0.5, up * K ** -0.5]


def both(x, residual, w, b):
    y, s = layer_norm(x, w, b, residual=residual)
    return y + s * 0.5


CALLS = {
    # a wave a row, a workgroup a row, and columns over several
    "norm": lambda: (tensors((5, 40), (40,), (40,)), lambda x, w, b: layer_norm(x, w, b)),
    "norm and stream": lambda: (tensors((70, 4100), (70, 4100), (4100,), (4100,), dtype=torch.bfloat16), both),
    "norm of wide rows": lambda: (tensors((9, 17000), (17000,), (17000,), dtype=torch.float16),
                                  lambda x, w, b: layer_norm(x, w, b)),
    "gated": lambda: (gated_leaves(130, 64, 200, torch.bfloat16), gated_linear),
    "gated, a factor": lambda: (gated_leaves(130, 64, 200, torch.float16), gated_linear),
    "gated, copies": lambda: (gated_leaves(70, 67, 3001, torch.bfloat16), gated_linear),
    "gated in fp32": lambda: (gated_leaves(40, 36, 50, torch.float32), gated_linear),
    "gated, parts": lambda: (gated_leaves(2000, 130, 1100, torch.float32), gated_linear),
}
NAMES = list(CALLS)


def step(f, leaves, up=None):
    leaves = [t.detach().requires_grad_() for t in leaves]
    out = f(*leaves)
    return [out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out) if up is None else up)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b, strict=True))


@pytest.mark.parametrize("name", NAMES)
def test_captured_steps(name):
    """A graph of a whole step, replayed with new inputs between eager work."""
    static, f = CALLS[name]()
    up = torch.ones_like(f(*static))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(f, static, up)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(f, static, up)
    for r in range(4):
        new = [t.roll(r + 1, 0) * 0.75 for t in static]
        up.copy_(torch.randn_like(up))
        want = step(f, new, up)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert same(res, want), f"replay {r}"


@pytest.mark.parametrize("name", NAMES)
def test_captured_forward_alone(name):
    """As serving does; two graphs of one call, replayed in turn."""
    static, f = CALLS[name]()
    with torch.no_grad():
        f(*static)
        graphs, res = [], []
        for _ in range(2):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                res.append(f(*static))
        for r in range(3):
            for a in static:
                a.copy_(a.roll(1, 0) * 0.9)
            want = f(*static)
            for g in graphs:
                g.replay()
            torch.cuda.synchronize()
            assert same(res, [want, want]), f"replay {r}"


@pytest.mark.parametrize("name", NAMES)
def test_on_other_streams_at_once(name):
    leaves, f = CALLS[name]()
    more = [t.flip(0) * 0.5 for t in leaves]
    want = [step(f, leaves), step(f, more)]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in sides:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        got = []
        for st, ts in zip(sides, (leaves, more)):
            with torch.cuda.stream(st):
                got.append(step(f, ts))
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", NAMES)
def test_no_gradient_of_a_gradient(name):
    leaves, f = CALLS[name]()
    leaves = [t.requires_grad_() for t in leaves]
    grads = torch.autograd.grad(f(*leaves).float().square().sum(), leaves, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        sum(g.float().square().sum() for g in grads).backward()


@pytest.mark.parametrize("name", NAMES)
def test_backward_twice_gives_the_same_bits(name):
    leaves, f = CALLS[name]()
    leaves = [t.requires_grad_() for t in leaves]
    out = f(*leaves)
    go = torch.ones_like(out)
    first = torch.autograd.grad(out, leaves, go, retain_graph=True)
    assert same(first, torch.autograd.grad(out, leaves, go))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, leaves, go)


@pytest.mark.parametrize("name,which", [("norm", 0), ("norm", 1), ("gated", 0), ("gated", 1),
                                        ("gated, a factor", 2)])
def test_a_changed_input_is_noticed(name, which):
    leaves, f = CALLS[name]()
    bases = [t.requires_grad_() for t in leaves]
    leaves = [t * 1.0 for t in bases]
    out = f(*leaves)
    with torch.no_grad():
        leaves[which].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("name", NAMES)
def test_saved_tensors_may_be_kept_elsewhere(name):
    leaves, f = CALLS[name]()
    want = step(f, leaves)[1:]
    leaves = [t.requires_grad_() for t in leaves]
    with torch.autograd.graph.save_on_cpu():
        out = f(*leaves)
    assert same(torch.autograd.grad(out, leaves, torch.ones_like(out)), want)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_a_trace_runs_the_kernels(name, train):
    leaves, f = CALLS[name]()
    leaves = [t.requires_grad_(train) for t in leaves]
    traced = torch.jit.trace(lambda *t: f(*t) * 2.0, leaves)
    for _ in range(2):
        leaves = [(t.detach().flip(0) * 0.5 + 0.25).requires_grad_(train) for t in leaves]
        want, got = f(*leaves) * 2.0, traced(*leaves)
        assert torch.equal(got, want)
        if train:
            ups = torch.ones_like(want)
            assert same(torch.autograd.grad(got, leaves, ups), torch.autograd.grad(want, leaves, ups))


@pytest.mark.parametrize("trains", [False, True])
@pytest.mark.parametrize("name", ["norm", "norm and stream", "gated"])
def test_tangents_are_refused(name, trains):
    leaves, f = CALLS[name]()
    for n in range(len(leaves)):
        with forward_ad.dual_level():
            given = [t.detach().clone().requires_grad_(trains) for t in leaves]
            given[n] = forward_ad.make_dual(given[n], torch.ones_like(given[n]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(*given)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                f(*given)
    f(*leaves)  # and none is left behind


@pytest.mark.parametrize("name", ["norm", "norm and stream", "gated"])
def test_double_precision_is_refused(name):
    leaves, f = CALLS[name]()
    with pytest.raises(RuntimeError, match="not implemented"):
        f(*(t.double() for t in leaves))


def test_refusals_on_the_gpu_are_the_checks_own():
    x, w, wide = tensors((4, 24), (24,), (4, 25))
    gate, short = tensors((8, 24), (7, 24))
    for error, match, f in (
            (ValueError, "weight must be", lambda: layer_norm(x, wide[0])),
            (ValueError, "residual must be", lambda: layer_norm(x, w, residual=wide)),
            (ValueError, "residual must be", lambda: layer_norm(x, w, residual=x[:1])),
            (ValueError, "weight must have dtype", lambda: layer_norm(x, w.half())),
            (ValueError, "weight", lambda: layer_norm(x, w.cpu())),
            (ValueError, "eps", lambda: layer_norm(x, w, eps=-1.0)),
            (ValueError, "eps", lambda: layer_norm(x, w, eps=float("nan"))),
            (ValueError, "eps", lambda: layer_norm(x, w, eps=float("inf"))),
            (TypeError, "floating point", lambda: layer_norm(x.int())),
            (ValueError, "width", lambda: layer_norm(x[0, 0])),
            (ValueError, "both be", lambda: gated_linear(x, gate, short)),
            (ValueError, "both be", lambda: gated_linear(wide, gate, gate)),
            (ValueError, "both be", lambda: gated_linear(x, gate[0], gate[0])),
            (ValueError, "up_weight must have dtype", lambda: gated_linear(x, gate, gate.half())),
            (ValueError, "up_weight", lambda: gated_linear(x, gate, gate.cpu())),
            (ValueError, "activation", lambda: gated_linear(x, gate, gate, activation="tanh")),
    ):
        with pytest.raises(error, match=match):
            f()


def test_widths_beyond_the_kernels_are_refused():
    x = torch.zeros(2, (1 << 20) + 8, device=DEV, dtype=torch.float16)
    w = torch.zeros(1, (1 << 20) + 8, device=DEV, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="2\\^20"):
        gated_linear(x, w, w)
    w.requires_grad_()
    with pytest.raises(RuntimeError, match="2\\^20"):
        gated_linear(x, w, w)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_share_memory_and_gradients_that_are_one_number(dtype):
    """An expanded x (rows of one token), overlapping rows, an upstream gradient of
    stride zero, as a sum's is."""
    K, F, M = 48, 40, 70
    line, gate, up, w = tensors((200 + K,), (F, K), (F, K), (K,), dtype=dtype)
    gate, up = gate / 7, up / 7
    for x in (line[None, :K].expand(M, K), line.as_strided((M, K), (1, 1)), line.as_strided((M, K), (2, 1)),
              line.as_strided((7, 10, K), (0, 8, 1)), line.as_strided((M, K), (1, 3))):
        flat = x.reshape(M, K).clone()
        vals, tols = oracle.gated(flat.cpu(), gate.cpu(), up.cpu(), "silu", torch.ones(M, F, dtype=dtype))
        leaf = [t.detach().requires_grad_() for t in (x, gate, up)]
        h = gated_linear(*leaf)
        got = torch.autograd.grad(h.sum(), leaf)
        oracle.close(h.view(M, F), vals["h"], tols["h"], "h")
        for v, n in zip(got, ("gx", "ggate", "gup")):
            oracle.close(v.reshape(vals[n].shape), vals[n], tols[n], n)
        vals, tols = oracle.layer_norm(flat.cpu(), w.cpu(), None, None, 1e-5, torch.ones(M, K, dtype=dtype))
        leaf = [t.detach().requires_grad_() for t in (x, w)]
        y = layer_norm(*leaf)
        gx, gw = torch.autograd.grad(y.sum(), leaf)
        oracle.close(y.view(M, K), vals["y"], tols["y"], "y")
        oracle.close(gx.reshape(M, K), vals["gx"], tols["gx"], "gx")
        oracle.close(gw, vals["gw"], tols["gw"], "gw")


def test_a_residual_of_other_strides_and_the_same_tensor_twice():
    (x, w) = tensors((6, 5, 24), (24,), dtype=torch.bfloat16)
    other = x.transpose(0, 1).contiguous().transpose(0, 1) * 2
    y, s = layer_norm(x, w, residual=other)
    vals, tols = oracle.layer_norm(x.view(30, 24).cpu(), w.cpu(), None, other.reshape(30, 24).cpu(), 1e-5)
    oracle.close(y.view(30, 24), vals["y"], tols["y"], "y")
    assert torch.equal(s, x + other) and s.is_contiguous()
    leaf = x.clone().requires_grad_()
    y, s = layer_norm(leaf, w, residual=leaf)
    (g,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    doubled = (x * 2).requires_grad_()
    (want,) = torch.autograd.grad(layer_norm(doubled, w), doubled, torch.ones_like(y))
    assert torch.equal(g, want * 2)


@pytest.mark.parametrize("name", ["norm", "gated in fp32", "gated, parts"])
def test_gradients_against_differences(name):
    """The kernels' gradient along a direction and the 64-bit forms' central difference:
    off by the gradients' own tolerances, and by the difference's cut-off series, a third
    of what a step of twice the length changes (a tenth of the result's last bits over the
    step is counted too)."""
    leaves, f = CALLS[name]()
    leaves = [t.cpu() for t in leaves]
    out = f(*(t.to(DEV) for t in leaves))
    up = torch.randn(out.shape, generator=torch.Generator().manual_seed(5))
    dirs = [torch.randn(t.shape, generator=torch.Generator().manual_seed(6)) for t in leaves]
    got = step(f, [t.to(DEV) for t in leaves], up.to(DEV))[1:]
    if name == "norm":
        vals, tols = oracle.layer_norm(*leaves, None, 1e-5, up)
        names = ("gx", "gw", "gb")
    else:
        vals, tols = oracle.gated(*leaves, "silu", up)
        names = ("gx", "ggate", "gup")
    along = sum(float((g.double().cpu() * d.double()).sum()) for g, d in zip(got, dirs))
    tol = sum(float((tols[n] * d.double().abs()).sum()) for n, d in zip(names, dirs))

    def loss(by):
        return float((f(*(t.double() + by * d.double() for t, d in zip(leaves, dirs))) * up.double()).sum())

    def difference(by):
        return (loss(by) - loss(-by)) / (2 * by)

    h = 2.0 ** -12
    near, far = difference(h), difference(2 * h)
    last = abs(loss(0.0)) * 2.0 ** -52 * 1e3 / h + 1e-9
    assert abs(along - near) <= tol + abs(far - near) + last


def test_large_offsets_of_the_gated_projections():
    """More than 2^31 elements of h and what stands behind it: the last rows, and the weights'
    gradients from them alone."""
    M, K, F = (1 << 31) // 16384 + 70, 16, 16384
    x, gate, up = gated_leaves(200, K, F, torch.bfloat16)
    x = torch.cat((torch.ones(M - 200, K, device=DEV, dtype=torch.bfloat16), x))
    leaf = [t.requires_grad_() for t in (x, gate, up)]
    h = gated_linear(*leaf)
    gh = torch.zeros_like(h)
    gh[-100:] = tensors((100, F), dtype=torch.bfloat16, seed=4)[0]
    got = torch.autograd.grad(h, leaf, gh)
    vals, tols = oracle.gated(x[-100:].detach().cpu(), gate.detach().cpu(), up.detach().cpu(), "silu", gh[-100:].cpu())
    oracle.close(h[-100:], vals["h"], tols["h"], "h")
    oracle.close(got[0][-100:], vals["gx"], tols["gx"], "gx")
    assert not got[0][:-100].any()
    oracle.close(got[1], vals["ggate"], tols["ggate"], "ggate")
    oracle.close(got[2], vals["gup"], tols["gup"], "gup")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_offsets_of_x(dtype):
    """More than 2^31 elements of x, in fp32 with copies in parts."""
    M, K, F = (1 << 31) // 2048 + 70, 2048, 24
    xs, gate, up = gated_leaves(100, K, F, dtype)
    x = torch.zeros(M, K, device=DEV, dtype=dtype)
    x[-100:] = xs
    leaf = [t.requires_grad_() for t in (x, gate, up)]
    h = gated_linear(*leaf)
    gh = torch.zeros_like(h)
    gh[-100:] = tensors((100, F), dtype=dtype, seed=4)[0]
    got = torch.autograd.grad(h, leaf, gh)
    vals, tols = oracle.gated(xs.cpu(), gate.detach().cpu(), up.detach().cpu(), "silu", gh[-100:].cpu())
    oracle.close(h[-100:], vals["h"], tols["h"], "h")
    assert not h[:-100].any()
    oracle.close(got[0][-100:], vals["gx"], tols["gx"], "gx")
    oracle.close(got[1], vals["ggate"], tols["ggate"], "ggate")
    oracle.close(got[2], vals["gup"], tols["gup"], "gup")


def test_large_offsets_of_the_norm():
    M, n = (1 << 31) // 2048 + 70, 2048
    xs, w, b, gs = tensors((100, n), (n,), (n,), (100, n), dtype=torch.bfloat16)
    x = torch.zeros(M, n, device=DEV, dtype=torch.bfloat16)
    x[-100:] = xs
    leaf = [t.requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaf)
    gy = torch.zeros_like(y)
    gy[-100:] = gs
    got = torch.autograd.grad(y, leaf, gy)
    vals, tols = oracle.layer_norm(xs.cpu(), w.detach().cpu(), b.detach().cpu(), None, 1e-5, gs.cpu())
    oracle.close(y[-100:], vals["y"], tols["y"], "y")
    assert torch.equal(y[:-100], b.detach().expand(M - 100, n))
    oracle.close(got[0][-100:], vals["gx"], tols["gx"], "gx")
    assert not got[0][:-100].any()
    oracle.close(got[1], vals["gw"], tols["gw"], "gw")
    oracle.close(got[2], vals["gb"], tols["gb"], "gb")


@pytest.mark.parametrize("dtype,M,K,F", [
    (torch.bfloat16, 1, 64, 160), (torch.float16, 40, 64, 160), (torch.bfloat16, 300, 136, 400),
    (torch.float16, 129, 67, 91), (torch.float32, 260, 64, 160)])
def test_a_blocks_second_half(dtype, M, K, F):
    """The norm of the stream, the gated projections (the halves of one matrix) and the last
    projection, added to the stream and normalized again: each operator against the formulas
    of what it was given, forward and backward, and a captured step against the eager one."""
    x, stream, both, down, w, b = tensors((M, K), (M, K), (2 * F, K), (K, F), (K,), (K,), dtype=dtype)
    leaves = [x, stream, both * K ** -0.5, down * F ** -0.5, w, b]

    def run(leaves, keep=lambda *t: None):
        x, stream, both, down, w, b = leaves
        y, s = layer_norm(x, w, b, residual=stream)
        h = gated_linear(y, both[:F], both[F:], activation="gelu_tanh")
        o = torch.nn.functional.linear(h, down)
        y2, s2 = layer_norm(o, w, b, residual=s)
        keep(y, s, h, o, y2, s2)
        return y2 + s2

    leaf = [t.clone().requires_grad_() for t in leaves]
    seen = []

    def keep(*t):
        seen.extend(t)
        for v in t:
            v.retain_grad()

    out = run(leaf, keep)
    up = tensors((M, K), dtype=dtype, seed=9)[0]
    grads = torch.autograd.grad(out, leaf + seen, up)
    y, s, h, o, y2, s2 = (t.detach().cpu() for t in seen)
    gy, gs, gh, go, gy2, gs2 = (t.cpu() for t in grads[6:])
    x, stream, both, down, w, b = (t.cpu() for t in leaves)

    vals, tols = oracle.gated(y, both[:F], both[F:], "gelu_tanh", gh)
    oracle.close(h, vals["h"], tols["h"], "h")
    oracle.close(gy, vals["gx"], tols["gx"], "gy")
    oracle.close(grads[2][:F], vals["ggate"], tols["ggate"], "gate")
    oracle.close(grads[2][F:], vals["gup"], tols["gup"], "up")
    second, second_tol = oracle.layer_norm(o, w, b, s, 1e-5, gy2, gs2)
    oracle.close(y2, second["y"], second_tol["y"], "y2")
    oracle.close(go, second["gx"], second_tol["gx"], "go")
    assert torch.equal(s2, second["s"].to(dtype))
    # (the stream's gradient: that of s2's sum, whose other side is o)
    assert torch.equal(gs, go)
    first, first_tol = oracle.layer_norm(x, w, b, stream, 1e-5, gy, gs)
    oracle.close(y, first["y"], first_tol["y"], "y")
    oracle.close(grads[0].cpu(), first["gx"], first_tol["gx"], "gx")
    assert torch.equal(grads[0], grads[1])
    for i, n in ((4, "gw"), (5, "gb")):  # both norms', added up in the type
        u = oracle.half_ulp(dtype)
        want = first[n] + second[n]
        tol = first_tol[n] + second_tol[n]
        oracle.close(grads[i], want, tol + u * (want.abs() + tol) + oracle.tiny(dtype), n)

    static = [t.clone() for t in leaves]

    def whole(ts):
        ts = [t.detach().requires_grad_() for t in ts]
        out = run(ts)
        return [out.detach(), *torch.autograd.grad(out, ts, up)]

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        whole(static)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = whole(static)
    for r in range(3):
        for t in static:
            t.copy_(t.roll(1, 0))
        want = whole(static)
        graph.replay()
        torch.cuda.synchronize()
        assert same(res, want), f"replay {r}"


def test_more_rows_than_workgroups():
    """A workgroup a row, as far as a launch's threads go: the last rows are those of a
    workgroup's second turn."""
    M, n = (1 << 21) + 300, 2056
    xs, w = tensors((300, n), (n,), dtype=torch.bfloat16)
    x = torch.ones(M, n, device=DEV, dtype=torch.bfloat16)
    x[-300:] = xs
    y = layer_norm(x, w)
    vals, tols = oracle.layer_norm(xs.cpu(), w.cpu(), None, None, 1e-5)
    oracle.close(y[-300:], vals["y"], tols["y"], "y")
    assert not y[:-300].any()


def test_rows_wider_than_a_launch_of_their_columns():
    """The weights' sums are taken 32 columns a workgroup, and again behind 2^25 of them."""
    n = (1 << 25) + 70
    x, gy = torch.zeros(2, n, device=DEV, dtype=torch.float16), torch.zeros(2, n, device=DEV, dtype=torch.float16)
    x[0, :n // 2], x[0, n // 2:] = 1.0, -1.0  # mean 0, variance 1
    gy[:, -100:] = tensors((2, 100), dtype=torch.float16)[0]
    b = torch.zeros(n, device=DEV, dtype=torch.float16).requires_grad_()
    w = torch.ones(n, device=DEV, dtype=torch.float16).requires_grad_()
    y = layer_norm(x, w, b, eps=0.0625)
    assert (y[0, n // 2:] == y[0, -1]).all() and abs(float(y[0, -1]) + 1.0625 ** -0.5) < 1e-3 and not y[1].any()
    gw, gb = torch.autograd.grad(y, [w, b], gy)
    want = gy[0, -100:].double() * -1.0625 ** -0.5
    assert (gw[-100:].double() - want).abs().max() <= 2.0 ** -9 * want.abs().max() and not gw[:-100].any()
    total = gy[:, -100:].double().sum(0)
    assert ((gb[-100:].double() - total).abs() <= 2.0 ** -11 * total.abs() + 2.0 ** -24).all() and not gb[:-100].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_gradients_of_a_row_without_numbers(dtype, bad):
    x, gate, up = gated_leaves(70, 64, 96, dtype)
    gh = tensors((70, 96), dtype=dtype, seed=8)[0]
    vals, tols = oracle.gated(x.cpu(), gate.cpu(), up.cpu(), "silu", gh.cpu())
    x[33, 5] = bad
    leaf = [t.requires_grad_() for t in (x, gate, up)]
    gx, gg, gu = torch.autograd.grad(gated_linear(*leaf), leaf, gh)
    assert gx[33].isnan().all() and gg[:, 5].isnan().all() and not gu[:, 5].isfinite().any()
    rest = [m for m in range(70) if m != 33]
    oracle.close(gx[rest], vals["gx"][rest], tols["gx"][rest], "gx")


def test_more_rows_than_a_launch_has_threads():
    """2^30 rows: 64 of them a workgroup would be a launch of 2^32 threads."""
    M, K, F = 1 << 30, 8, 1
    xs, gate, up = gated_leaves(100, K, F, torch.bfloat16)
    x = torch.zeros(M, K, device=DEV, dtype=torch.bfloat16)
    x[-100:] = xs
    h = gated_linear(x, gate, up)
    vals, tols = oracle.gated(xs.cpu(), gate.cpu(), up.cpu(), "silu")
    oracle.close(h[-100:], vals["h"], tols["h"], "h")
    assert not h[:-100].any()
    with pytest.raises(RuntimeError, match="2\\^30"):
        gated_linear(torch.zeros(1, K, device=DEV, dtype=torch.bfloat16).expand(M + 1, K), gate, up)


def test_gradients_of_more_blocks_than_workgroups():
    """dg and du of 2^25 rows and some: workgroups take turns."""
    M, K, F = (1 << 25) + 100, 8, 16
    xs, gate, up = gated_leaves(100, K, F, torch.bfloat16)
    x = torch.zeros(M, K, device=DEV, dtype=torch.bfloat16)
    x[-100:] = xs
    leaf = [t.requires_grad_() for t in (x, gate, up)]
    h = gated_linear(*leaf)
    gh = torch.zeros_like(h)
    gh[-100:] = tensors((100, F), dtype=torch.bfloat16, seed=4)[0]
    got = torch.autograd.grad(h, leaf, gh)
    vals, tols = oracle.gated(xs.cpu(), gate.detach().cpu(), up.detach().cpu(), "silu", gh[-100:].cpu())
    for v, n in zip((h, *got), ("h", "gx", "ggate", "gup")):
        oracle.close(v[-100:], vals[n], tols[n], n)
    assert not got[0][:-100].any()


def test_a_conjugates_imaginary_part():
    """A real tensor whose numbers lie in memory with the other sign."""
    a = tensors((40, 1))[0]
    x = torch.complex(a, a).conj().imag
    assert x.is_neg()
    w = tensors((8, 1), seed=4)[0]
    assert torch.equal(gated_linear(x, w, w), gated_linear(-a, w, w))
    y, s = layer_norm(x, residual=x)
    assert torch.equal(s, -2 * a) and not y.any()


@pytest.mark.parametrize("dtype,n", [("bf16", 4104), ("bf16", 4099), ("fp16", 16001), ("fp16", 12000), ("fp32", 2051),
                                     ("fp32", 8188), ("bf16", 17003)])
def test_rows_that_workgroups_walk(dtype, n):
    """Three rows and more a workgroup of 512, forward and backward, with the loads of the
    next ones under way, and rows that are read again."""
    check_norm(norm_inputs(1700, n, dtype, residual=n % 2 == 0))

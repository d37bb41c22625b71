"""The gated projections in fp32 as sums of six products of bf16 parts: that none of the six
is lost in h or in a gradient.  What each test's inputs would show is itself tested on the CPU,
by leaving products out."""
from __future__ import annotations

import pytest
import torch

from neural_shift_cuda import gated_linear

DEV = "cuda"
M, K, F = 2000, 132, 1100  # sizes that are taken apart (test_gpu_gated_parts.py)
SIX = [(2, 0), (0, 2), (1, 1), (1, 0), (0, 1), (0, 0)]

# Whole numbers that need two and three parts of 8 bits.  Sums of up to 250 products of two of the
# first kind, or of the second and 1, stay below 2^24: exact in any order.
TWO, THREE = 2 ** 8 + 1, 2 ** 16 + 2 ** 8 + 1
SIDES = {"two by two": (TWO, TWO, [(0, 0), (1, 0), (0, 1), (1, 1)]),
         "three by one": (THREE, 1, [(0, 0), (1, 0), (2, 0)]),
         "one by three": (1, THREE, [(0, 0), (0, 1), (0, 2)])}


def signs(*shape, seed=0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    return torch.randint(0, 2, shape, generator=g).float() * 2 - 1


def sparse(t, most, dim):
    """`most` of t along dim, here and there, and zeros."""
    g = torch.Generator().manual_seed(11)
    keep = torch.rand(t.shape, generator=g).argsort(dim).argsort(dim) < most
    return t * keep


def full(*shape, seed):
    """Numbers of 24 bits in [1, 2)."""
    return 1.0 + torch.rand(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64).float()


# Every case: (x, gate, up, gh), which result is looked at (and its columns), what it has to be, and
# the two matrices whose product it is (rows by contraction each).  relu, and the gate 1 (or the
# other projection 1) where the product is not its own.
def value_case(a, b, side):
    x, w = a.clone(), b.clone()
    x[:, 0], w[:, 0] = 1.0, 0.0
    one = torch.zeros(F, K)
    one[:, 0] = 1.0
    want = x.double() @ w.double().t()
    if side == "gate":
        return (x, w, one, torch.zeros(M, F)), "h", slice(None), want.clamp_min(0), (x, w)
    return (x, one, w, torch.zeros(M, F)), "h", slice(None), want, (x, w)


def input_case(d, gate, up):
    gate, up = gate.clone(), up.clone()
    gate[:, 0] = up[:, 0] = 1.0
    x = torch.zeros(M, K)
    x[:, 0] = 1.0
    both, two = torch.cat((gate, up)), torch.cat((d, d), 1)
    return (x, gate, up, d), "gx", slice(1, None), (two.double() @ both.double())[:, 1:], (two, both.t()[1:])


def weight_case(d, x, which):
    x = x.clone()
    x[:, 0] = 1.0
    one = torch.zeros(F, K)
    one[:, 0] = 1.0
    return (x, one, one, d), which, slice(1, None), (d.double().t() @ x.double())[:, 1:], (d.t(), x.t()[1:])


def whole_number_cases(kind):
    p, q, _ = SIDES[kind]
    yield value_case(p * signs(M, K), q * signs(F, K), "gate")
    yield value_case(p * signs(M, K), q * signs(F, K, seed=1), "up")
    yield input_case(p * sparse(signs(M, F), 100, 1), q * signs(F, K), q * signs(F, K, seed=1))
    for which in ("ggate", "gup"):
        yield weight_case(p * sparse(signs(M, F), 200, 0), q * signs(M, K), which)


def single_product_cases():
    yield value_case(sparse(full(M, K, seed=1), 0, 1) + torch.nn.functional.pad(full(M, 1, seed=1), (5, K - 6)),
                     full(F, K, seed=2), "gate")
    yield value_case(torch.nn.functional.pad(full(M, 1, seed=1), (5, K - 6)), full(F, K, seed=3), "up")
    yield input_case(sparse(full(M, F, seed=4), 1, 1), full(F, K, seed=5), torch.zeros(F, K))
    for which in ("ggate", "gup"):
        yield weight_case(sparse(full(M, F, seed=6), 1, 0), full(M, K, seed=7), which)


def run(x, gate, up, gh):
    leaves = [t.to(DEV).requires_grad_() for t in (x, gate, up)]
    h = gated_linear(*leaves, activation="relu")
    return dict(zip(("h", "gx", "ggate", "gup"), (h.detach(), *torch.autograd.grad(h, leaves, gh.to(DEV)))))


# ---------------------------------------------------------------------------
# On the CPU: what leaving a product out would do
# ---------------------------------------------------------------------------

def split(x):
    """Three parts of 8 bits each, all of x's sign."""
    parts, rest = [], x
    for _ in range(3):
        p = (rest.contiguous().view(torch.int32) & -65536).view(torch.float32)
        parts.append(p.double())
        rest = rest - p
    assert not rest.any()
    return parts


def by_parts(first, second, terms):
    p, q = split(first), split(second)
    return sum(p[i] @ q[j].t() for i, j in terms)


@pytest.mark.parametrize("kind", list(SIDES))
def test_whole_numbers_show_every_product(kind):
    for _, name, cols, want, (a, b) in whole_number_cases(kind):
        a, b = a[:64], b[:64]
        assert torch.equal(by_parts(a, b, SIX), a.double() @ b.double().t())
        assert (a.double().abs() @ b.double().abs().t()).max() < 2 ** 24
        for lost in SIDES[kind][2]:
            left = by_parts(a, b, [t for t in SIX if t != lost])
            assert not torch.equal(left, by_parts(a, b, SIX)), (name, lost)
    assert {t for k in SIDES for t in SIDES[k][2]} == set(SIX)


def test_single_products_show_every_product():
    for _, name, _, want, (a, b) in single_product_cases():
        exact = a[:200].double() @ b[:200].double().t()
        some = exact != 0

        def off(terms):
            return float(((by_parts(a[:200], b[:200], terms) - exact)[some] / exact[some]).abs().max())

        assert some.any() and off(SIX) <= 2.0 ** -21
        for lost in SIX:
            assert off([t for t in SIX if t != lost]) > 2.0 ** -18, (name, lost)


# ---------------------------------------------------------------------------
# The kernels
# ---------------------------------------------------------------------------

def looked_at(got, name, cols):
    return got[name].cpu().double()[:, cols]


@pytest.mark.parametrize("kind", list(SIDES))
@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_whole_numbers_are_exact(kind):
    for inputs, name, cols, want, _ in whole_number_cases(kind):
        assert torch.equal(looked_at(run(*inputs), name, cols), want), name


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
def test_single_products():
    """One product in a sum: the three that are left out are below 2^-21 of it (a second part is
    below 2^-7 and a third below 2^-15), and six additions and a product round, of which all but
    two are of 2^-6 of it and less."""
    for inputs, name, cols, want, _ in single_product_cases():
        got = looked_at(run(*inputs), name, cols)
        assert not got[want == 0].any()
        off = float(((got - want)[want != 0] / want[want != 0]).abs().max())
        assert off <= 2.0 ** -20, (name, off)

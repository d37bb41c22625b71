"""Layer norm and the gated projections in 64 bits on the CPU, written from their
formulas, and how far a computation in fp32 with operands and results of a
narrower type may be from them.

A rounding to type t is off by at most u = eps(t) / 2 of the value; a sum of fp32
numbers by at most its longest chain of additions times 2^-24 of the sum of their
magnitudes.
"""
from __future__ import annotations

import math

import torch

from token_oracle import F32, close, half_ulp, tiny  # noqa: F401


def layer_norm(x, weight, bias, residual, eps, gy=None, gs=None):
    """(values, tolerances) by name of rows x (M, n): y, s and, with gy, gx, gw, gb."""
    u, least = half_ulp(x.dtype), tiny(x.dtype)
    M, n = x.shape
    # a lane adds up at most 32 columns in a row (or n / 1024 of them, eight at a time),
    # then lanes and waves meet in at most 24 steps
    k = (64 + n / 128) * F32
    vals, tols = {}, {}
    s = x
    if residual is not None:
        s = (x.float() + residual.float()).to(x.dtype)
        vals["s"], tols["s"] = s.double(), torch.zeros(())
    S = s.double()
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(n, dtype=torch.float64) if bias is None else bias.double()
    mean = S.mean(-1, keepdim=True)
    d = S - mean
    var = d.square().mean(-1, keepdim=True)
    r = (var + eps) ** -0.5
    h = d * r
    off = k * S.abs().mean(-1, keepdim=True)         # of the mean
    eh = off * r + h.abs() * (k + 4 * F32 + off.square() * r * r)
    vals["y"] = h * w + b
    tols["y"] = u * vals["y"].abs() + eh * w.abs() + 4 * F32 * (h * w).abs() \
        + 2 * F32 * vals["y"].abs() + least
    if gy is not None:
        g = gy.double()
        t = g * w
        m1, m2 = t.mean(-1, keepdim=True), (t * h).mean(-1, keepdim=True)
        core = r * (t - m1 - h * m2)
        vals["gx"] = core + (0 if gs is None else gs.double())
        size = t.abs() + t.abs().mean(-1, keepdim=True) + h.abs() * (t * h).abs().mean(-1, keepdim=True)
        off_r = k + 4 * F32 + off.square() * r * r
        tols["gx"] = u * vals["gx"].abs() + 2 * F32 * vals["gx"].abs() + least \
            + r * ((k + 8 * F32) * size + eh * m2.abs() + h.abs() * (t.abs() * eh).mean(-1, keepdim=True)) \
            + core.abs() * off_r
        vals["gw"], vals["gb"] = (g * h).sum(0), g.sum(0)
        chain = (M + 8) * F32
        tols["gw"] = u * vals["gw"].abs() + chain * (g * h).abs().sum(0) + (g.abs() * eh).sum(0) + least
        tols["gb"] = u * vals["gb"].abs() + chain * g.abs().sum(0) + least
    return vals, tols


def activation(kind, g):
    """Value and slope."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if kind == "gelu":
        below = 0.5 * torch.special.erfc(-g / math.sqrt(2))
        return g * below, below + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        a, b = math.sqrt(2 / math.pi), 0.044715
        t = torch.tanh(a * (g + b * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * a * (1 + 3 * b * g * g)
    if kind == "relu":
        return g.clamp_min(0), (g > 0).double()
    s = torch.sigmoid(g)
    return s, s * (1 - s)


def gated(x, gate, up, kind, gh=None):
    """(values, tolerances) by name of rows x (M, K): h and, with gh, gx, ggate and gup."""
    u_t, least = half_ulp(x.dtype), tiny(x.dtype)
    X, G, U = x.double(), gate.double(), up.double()
    K, F = G.shape[1], G.shape[0]
    g, u = X @ G.t(), X @ U.t()
    # K products and as many additions of fp32, each of them rounded or cut off
    k = 2 * (2 * K + 4) * F32
    eg, eu = k * (X.abs() @ G.abs().t()), k * (X.abs() @ U.abs().t())
    a, slope = activation(kind, g)
    # the exponentials' arguments are rounded: up to their size in steps; slopes of the
    # activations are at most 1.13, and change by at most 1.2 a unit (relu's: at 0)
    fine = (32 + 16 * g.abs() + 4 * g.square() + 2 * g.abs() ** 3) * F32
    ea = 1.13 * eg + fine * a.abs()
    es = (1.0 * (g.abs() <= eg) if kind == "relu" else 1.2 * eg) + fine * (slope.abs() + a.abs()) + 1e-30
    h = a * u
    vals = {"h": h}
    tols = {"h": u_t * h.abs() + ea * u.abs() + a.abs() * eu + ea * eu + 4 * F32 * h.abs() + least + 1e-36}
    if gh is None:
        return vals, tols
    d = gh.double()
    s, es = u * slope, es * (u.abs() + eu) + slope.abs() * eu + 4 * F32 * (u * slope).abs()
    dg, du = d * s, d * a
    # rounded as operands (fp16 times a power of two: below 2^-37 of the largest nothing is kept)
    floor = 2.0 ** -37 * d.abs().max() * max(s.abs().max(), a.abs().max()) if x.dtype == torch.float16 else 0.0
    edg = d.abs() * es + u_t * (dg.abs() + d.abs() * es) + floor + 1e-36
    edu = d.abs() * ea + u_t * (du.abs() + d.abs() * ea) + floor + 1e-36
    chain = 2 * (4 * F + 8) * F32
    vals["gx"] = dg @ G + du @ U
    tols["gx"] = u_t * vals["gx"].abs() + edg @ G.abs() + edu @ U.abs() \
        + chain * (dg.abs() @ G.abs() + du.abs() @ U.abs()) + least
    chain = 2 * (2 * X.shape[0] + 4) * F32
    for name, t, e in (("ggate", dg, edg), ("gup", du, edu)):
        vals[name] = t.t() @ X
        tols[name] = u_t * vals[name].abs() + e.t() @ X.abs() + chain * (t.abs().t() @ X.abs()) + least
    return vals, tols


def close_on_average(got, want, dtype, roundings, what):
    """The whole's relative error: independent roundings of at most half a step, u / sqrt(3)
    each at the most, add in squares; a twentieth for what fp32 adds to them."""
    got, want = got.detach().double().cpu(), want.double()
    off = float((got - want).norm() / want.norm().clamp_min(1e-300))
    most = 1.05 * half_ulp(dtype) * math.sqrt(roundings / 3)
    assert off <= most, f"{what}: {off:.3g} of the whole, {most:.3g} for {roundings} roundings"

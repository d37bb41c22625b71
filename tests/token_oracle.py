"""The token operators in 64 bits on the CPU, dense and written from their
formulas, and how far a computation in fp32 with operands and results of a
narrower type may be from them.

A rounding to type t is off by at most u = eps(t) / 2 of the value; a sum of n
fp32 products by at most (n + 1) 2^-24 of the sum of their magnitudes.
"""
from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24
INF = math.inf


def half_ulp(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half a step of the type's smallest numbers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def close(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} for {tuple(want.shape)}"
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN elsewhere"
    inf = want.isinf() | got.isinf()
    assert torch.equal(got[inf], want[inf]), f"{what}: infinities elsewhere"
    ok = ~(inf | want.isnan())
    err, tol = (got - want).abs()[ok], tol.double().expand(want.shape)[ok]
    bad = err > tol
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{float((err / tol.clamp_min(1e-300)).max()):.3g} of the tolerance "
                           f"(err {float(err[bad].max()):.3g})")


# ---------------------------------------------------------------------------
# norm and rotation
# ---------------------------------------------------------------------------

def norm_rotary(x, w, cos, sin, positions, eps, interleaved, g=None):
    """(values, tolerances) by name: out and, with g, gx and gw (of one of the
    two tensors; positions (B, L))."""
    u, least = half_ulp(x.dtype), tiny(x.dtype)
    B, H, L, D = x.shape
    half = cos.shape[1]
    X, W = x.double(), (torch.ones(D) if w is None else w).double()
    R = torch.eye(D, dtype=torch.float64).repeat(B, L, 1, 1)
    for b in range(B):
        for t in range(L):
            for i in range(half):
                lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
                p = int(positions[b, t])
                c, s = (cos[p, i], sin[p, i]) if 0 <= p < cos.shape[0] else (math.nan, math.nan)
                R[b, t, lo, lo] = R[b, t, hi, hi] = c
                R[b, t, lo, hi], R[b, t, hi, lo] = -s, s
    R = R[:, None]
    r = (X.square().mean(-1, keepdim=True) + eps) ** -0.5

    def turned(M, y):
        # a NaN turns its own pair only, not the rest of the row through 0 * NaN
        out = torch.matmul(M.nan_to_num(0.0), y[..., None])[..., 0]
        return torch.where(M.isnan().any(-1), math.nan, out)

    out = turned(R, X * r * W)
    # sum of squares, root, two products, the turn: (D + 12) roundings of fp32
    k = (D + 12) * F32
    vals, tols = {"out": out}, {"out": u * out.abs() + k * turned(R.abs(), (X * r * W).abs())
                                + least}
    if g is not None:
        Rt = R.transpose(-1, -2)
        G = turned(Rt, g.double())
        Ga = turned(Rt.abs(), g.double().abs())
        gw = G * W
        dot = (gw * X).mean(-1, keepdim=True)
        vals["gx"] = r * (gw - X * r * r * dot)
        size = r * (Ga * W.abs() + X.abs() * r * r * (Ga * W.abs() * X.abs()).mean(-1, keepdim=True))
        tols["gx"] = u * vals["gx"].abs() + 3 * k * size + least
        vals["gw"] = (G * X * r).sum((0, 1, 2))
        n = B * H * L
        tols["gw"] = u * vals["gw"].abs() + (k + (n + 4) * F32) * (Ga * X.abs() * r).sum((0, 1, 2)) \
            + least
    return vals, tols


# ---------------------------------------------------------------------------
# position bias
# ---------------------------------------------------------------------------

def relative(Lq, Lk, n=None):
    n = Lk if n is None else n
    return torch.arange(Lk)[None] - (torch.arange(Lq)[:, None] + n - Lq)


def position_bias(table, buckets, Lq, Lk):
    R = (len(buckets) - 1) // 2
    out = torch.empty(table.shape[1], Lq, Lk, dtype=torch.float64)
    rel = relative(Lq, Lk)
    for i in range(Lq):
        for j in range(Lk):
            b = int(buckets[max(-R, min(R, int(rel[i, j]))) + R])
            out[:, i, j] = table[b].double() if 0 <= b < table.shape[0] else math.nan
    return out


def position_bias_grad(go, buckets, nb):
    R = (len(buckets) - 1) // 2
    H, Lq, Lk = go.shape
    ids = buckets.long()[relative(Lq, Lk).clamp(-R, R) + R]
    g, size = torch.zeros(nb, H, dtype=torch.float64), torch.zeros(nb, H, dtype=torch.float64)
    for b in range(nb):
        g[b] = (go.double() * (ids == b)).sum((1, 2))
        size[b] = (go.double().abs() * (ids == b)).sum((1, 2))
    u = half_ulp(go.dtype)
    # the longest chain of additions: a diagonal or a lane's part of the ends,
    # then the chunks, then the bucket's positions
    steps = Lq + Lk + 2 * R + 64
    return g, u * g.abs() + steps * F32 * size + tiny(go.dtype)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def visible(B, Lq, Lk, causal=False, prefix=None, documents=None, lengths=None):
    see = torch.zeros(B, Lq, Lk, dtype=torch.bool)
    for b in range(B):
        n = Lk if lengths is None else max(0, min(Lk, int(lengths[b])))
        for i in range(Lq):
            p = i + n - Lq
            for j in range(n):
                ok = not causal or j <= p or (prefix is not None and j < int(prefix[b]))
                if documents is not None:
                    own = int(documents[b, p]) if p >= 0 else -1
                    ok = ok and own >= 0 and int(documents[b, j]) == own
                see[b, i, j] = ok
    return see


def attention(q, k, v, *, scale=None, cap=None, causal=False, prefix=None, documents=None,
              lengths=None, slopes=None, bias_table=None, buckets=None, go=None, gdegree=None):
    """(values, tolerances) by name: out, degree and, with go, gq, gk, gv (and
    gtable with a bias table)."""
    dt = q.dtype
    u, least = half_ulp(dt), tiny(dt)
    B, Hq, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    per = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    see = visible(B, Lq, Lk, causal, prefix, documents, lengths)
    Q, K, V = q.double(), k.double().repeat_interleave(per, 1), v.double().repeat_interleave(per, 1)
    live = see.any(1)[:, None, :, None]  # keys that some query sees
    K, V = torch.where(live, K, 0.0), torch.where(live, V, 0.0)
    x = scale * Q @ K.transpose(2, 3)
    # errors of a score: the product's D + 2 roundings, the cap's (exp and
    # reciprocal of one part in 2^22 on a value of up to twice the cap), the
    # biases' and the sum's
    ex = (D + 4) * F32 * abs(scale) * (Q.abs() @ K.abs().transpose(2, 3))
    t = torch.tanh(x / cap) if cap else None
    s = cap * t if cap else x
    if cap:
        ex = ex + 16 * F32 * cap
    rel = torch.stack([relative(Lq, Lk, None if lengths is None else
                                max(0, min(Lk, int(lengths[b])))) for b in range(B)])
    if slopes is not None:
        lin = slopes.double()[:, None, None] * rel.abs()[:, None]
        s, ex = s - lin, ex + 4 * F32 * lin
    if bias_table is not None:
        R = (len(buckets) - 1) // 2
        ids = buckets.long()[rel.clamp(-R, R) + R]
        tb = bias_table.double()[ids].permute(0, 3, 1, 2)
        s = s + tb
        ex = ex + 4 * F32 * torch.where(tb.isinf(), 0.0, tb).abs()
    see = see[:, None].expand(s.shape) & (s != -INF)
    s = s.masked_fill(~see, -INF)
    degree = torch.logsumexp(s, -1)
    p = torch.exp(s - torch.where(degree == -INF, 0.0, degree)[..., None]).masked_fill(~see, 0.0)
    # a probability: its own score's error, the degree's (no more than the row's
    # largest, weighted), the exponential's and the sum's; scores far below the
    # row's top count with their probability
    size = torch.where(see, s.abs(), 0.0)
    es = torch.where(see, ex + 4 * F32 * size, 0.0)
    row = (p * es).sum(-1, keepdim=True) + (16 + Lk / 8) * F32
    ep = es + row
    out = p @ V
    vals = {"out": out, "degree": degree}
    pv = p @ V.abs()
    eo = u * out.abs() + u * pv + (p * ep) @ V.abs() + (Lk / 8 + 16) * F32 * pv + least
    # (probabilities below the type's smallest numbers are lost)
    eo = eo + tiny(dt) * V.abs().sum(2, keepdim=True)
    tols = {"out": eo, "degree": row.squeeze(-1) + 8 * F32 * torch.where(
        degree.isinf(), 0.0, degree).abs()}
    if go is None:
        return vals, tols
    G = go.double()
    gd = torch.zeros_like(degree) if gdegree is None else gdegree.double()
    dP = G @ V.transpose(2, 3)
    edP = (D + 2) * F32 * (G.abs() @ V.abs().transpose(2, 3))
    delta = (G * out).sum(-1) - gd
    edelta = (G.abs() * (eo + (D + 2) * F32 * out.abs())).sum(-1) + F32 * gd.abs()
    dS = p * (dP - delta[..., None])
    edS = p * (edP + edelta[..., None]) + ep * dS.abs() + 4 * F32 * p * (
        dP.abs() + delta.abs()[..., None])
    # probabilities a 16-bit type cannot hold, times what they multiply
    lost = tiny(dt)
    pg = p.transpose(2, 3) @ G
    pga = p.transpose(2, 3) @ G.abs()
    egv = u * pga + (p * ep).transpose(2, 3) @ G.abs() + (Lq / 8 + 16) * F32 * pga \
        + lost * G.abs().sum(2, keepdim=True)
    slope = scale * (1 - t * t) if cap else torch.full_like(s, scale)
    dX = dS * slope
    # the cap's derivative 1 - t^2 carries an absolute error of its own
    edX = edS * slope.abs() + (32 * F32 * abs(scale) if cap else 0) * dS.abs() \
        + (2 * es * abs(scale) / cap * dS.abs() if cap else 0)
    full = u * dX.abs() + edX + lost * see
    gq, egq = dX @ K, full @ K.abs() + (Lk / 8 + 16) * F32 * (dX.abs() @ K.abs())
    gk = dX.transpose(2, 3) @ Q
    egk = full.transpose(2, 3) @ Q.abs() + (Lq / 8 + 16) * F32 * (dX.abs().transpose(2, 3) @ Q.abs())

    def shared(y):
        return y.unflatten(1, (Hk, per)).sum(2)

    vals["gq"], tols["gq"] = gq, egq + u * gq.abs() + least
    for n, g, e in (("gk", gk, egk), ("gv", pg, egv)):
        vals[n] = shared(g)
        tols[n] = shared(e) + u * vals[n].abs() + per * F32 * shared(g.abs()) + least
    if bias_table is not None:
        gt, et, sz = (torch.zeros(bias_table.shape, dtype=torch.float64) for _ in range(3))
        for b in range(bias_table.shape[0]):
            at = (ids == b)[:, None]
            gt[b], et[b] = (dS * at).sum((0, 2, 3)), (edS * at).sum((0, 2, 3))
            sz[b] = (dS.abs() * at).sum((0, 2, 3))
        vals["gtable"] = gt
        tols["gtable"] = et + u * gt.abs() + (Lq + 2 * R + 64) * F32 * sz + least
    return vals, tols

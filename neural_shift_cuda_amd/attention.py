"""Token operators: attention over sequences of tokens, next to the shift
windows of ``ops.py`` (extensions, no counterpart in the reference).

    qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions=None, *,
        eps=1e-6, interleaved=False)                 -> (q', k')
    relative_position_bias(table, buckets, q_len, k_len)  -> (H, q_len, k_len)
    biased_attention(q, k, v, *, scale, cap, causal, prefix, documents,
        lengths, slopes, bias_table, buckets,
        return_log_degree=False)                     -> D or (D, log_C)

and the tables a program makes once: ``rotary_table``, ``relative_buckets``.

Tensors are (B, heads, tokens, width).  The conventions are those of the
normalized accumulation: D = sum_j a_j v_j / sum_j a_j with a = exp(score),
log_C the logarithm of the sum, and a row that sees nothing gives D = 0 and
log_C = -inf.  GPU tensors go through autograd nodes in C++
(host/token_calls.cpp) into the HIP library (fp16, bf16, fp32; sums, norms and
softmax statistics in fp32); CPU tensors use the ``*_reference`` implementations
(any floating type), which are also exported.  A GPU tensor never falls back to
them.

Where tokens stand: the Lq queries are the last of the n filled keys (n = Lk,
or ``lengths[b]``), so query i has position i + n - Lq.  A training step has
Lq = Lk, a single new token Lq = 1.
"""
from __future__ import annotations

import functools
import math
from typing import Optional, Tuple

import torch

from . import ops

_C = ops._C
_NEG_INF = float("-inf")
MAX_REACH = 2048  # relative positions a bucket map may tell apart, each way


# ---------------------------------------------------------------------------
# Tables a program makes once
# ---------------------------------------------------------------------------

def rotary_table(positions, dim: int, *, base: float = 10000.0, device=None
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(cos, sin), float32 (P, dim / 2), of the angles position * base^(-2 i / dim).

    `positions` is a count P (positions 0 .. P-1) or a tensor of P positions,
    or of (P, A) coordinates: the dim / 2 pairs are then shared out to the A axes
    in equal parts (image tokens: row and column).  The angles are formed in
    64 bits: in 32, position 10^5 is already 4e-3 rad off."""
    if isinstance(positions, int):
        positions = torch.arange(positions, device=device)
    if positions.dim() not in (1, 2):
        raise ValueError(f"positions must be a count, (P,) or (P, A); got {tuple(positions.shape)}")
    at = positions.to(device=device, dtype=torch.float64)
    at = at[:, None] if at.dim() == 1 else at
    axes = at.shape[1]
    if dim < 0 or dim % 2 or axes < 1 or (dim // 2) % axes:
        raise ValueError(f"dim must be even and its pairs divide among {axes} axes; got {dim}")
    part = dim // axes
    freq = base ** (-torch.arange(0, part, 2, dtype=torch.float64, device=at.device) / max(part, 1))
    angle = (at[:, :, None] * freq).flatten(1)
    return angle.cos().float(), angle.sin().float()


def relative_buckets(num_buckets: int, reach: int, *, bidirectional: bool = True, device=None
                     ) -> torch.Tensor:
    """int32 (2 * reach + 1): the bucket of each relative position (key minus
    query) from -reach to reach; those beyond share the ends' buckets.

    Half of the buckets are single distances, the others grow with the
    logarithm of the distance up to `reach`.  `bidirectional`: keys after the
    query have the second half of the buckets to themselves; otherwise they
    share bucket 0 with the query's own position."""
    n = num_buckets // 2 if bidirectional else num_buckets
    near = n // 2
    if near < 1 or not near < reach <= MAX_REACH:
        raise ValueError(f"relative_buckets needs num_buckets >= {4 if bidirectional else 2} and "
                         f"{near} < reach <= {MAX_REACH}; got {num_buckets}, {reach}")
    rel = torch.arange(-reach, reach + 1)
    d = rel.abs() if bidirectional else (-rel).clamp_min(0)
    far = near + (torch.log(d.clamp_min(near).double() / near) / math.log(reach / near)
                  * (n - near)).long()
    out = torch.where(d < near, d, far.clamp_max(n - 1))
    if bidirectional:
        out = out + n * (rel > 0)
    return out.to(device=device, dtype=torch.int32)


# ---------------------------------------------------------------------------
# Argument handling
# ---------------------------------------------------------------------------

def _heads(t: torch.Tensor, name: str) -> None:
    if t.dim() != 4:
        raise ValueError(f"{name} must be (B, heads, tokens, width); got {tuple(t.shape)}")
    if not t.is_floating_point():
        raise TypeError(f"{name} must be floating point; got {t.dtype}")


def _same(name: str, t: torch.Tensor, like: torch.Tensor, dtype: bool = True) -> None:
    if t.device != like.device:
        raise ValueError(f"{name} must be on {like.device}; got {t.device}")
    if dtype and t.dtype != like.dtype:
        raise ValueError(f"{name} must have dtype {like.dtype}; got {t.dtype}")


def _integers(name: str, t: torch.Tensor, shape, like: torch.Tensor) -> None:
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise TypeError(f"{name} must hold integers; got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)}; got {tuple(t.shape)}")
    _same(name, t, like, dtype=False)


def _whole(name: str, t: Optional[torch.Tensor], shape, like: torch.Tensor
           ) -> Optional[torch.Tensor]:
    """An integer tensor of a given shape as contiguous int32 (values beyond
    it at its ends: no row, bucket or length that the operators serve)."""
    if t is None:
        return None
    if t.dtype is torch.int32 and t.shape == shape and t.device == like.device:
        return t.contiguous()
    _integers(name, t, shape, like)
    if t.dtype == torch.uint64:  # the upper half has no place among the signed
        t = t.view(torch.int64)
        t = torch.where(t < 0, (1 << 31) - 1, t)
    elif t.dtype == torch.uint32:
        t = t.long()
    if t.dtype == torch.int64:
        t = t.clamp(-(1 << 31), (1 << 31) - 1)
    return t.to(torch.int32).contiguous()


def _documents(t: Optional[torch.Tensor], shape, like: torch.Tensor) -> Optional[torch.Tensor]:
    """Document numbers, contiguous: as int32, or, where the type holds more, as
    int64.  Only which are equal and which are negative counts, so no two may
    fall together as ``_whole`` lets them."""
    if t is None:
        return None
    _integers("documents", t, shape, like)
    if t.dtype == torch.uint64:  # numbered anew: the upper half would turn negative
        t = torch.unique(t.view(torch.int64), return_inverse=True)[1]
    wide = t.dtype in (torch.int64, torch.uint32)
    return t.to(torch.int64 if wide else torch.int32).contiguous()


def _acc(t: torch.Tensor) -> torch.dtype:
    return torch.float64 if t.dtype == torch.float64 else torch.float32


def _check_norm(q, k, q_weight, k_weight, cos, sin, positions):
    _heads(q, "q")
    _heads(k, "k")
    _same("k", k, q)
    B, _, L, D = q.shape
    if k.shape[0] != B or k.shape[2] != L or k.shape[3] != D:
        raise ValueError(f"q and k must agree but for their heads; got {tuple(q.shape)} and "
                         f"{tuple(k.shape)}")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None:
            _same(name, w, q)
            if tuple(w.shape) != (D,):
                raise ValueError(f"{name} must be ({D},); got {tuple(w.shape)}")
    for name, t in (("cos", cos), ("sin", sin)):
        _same(name, t, q, dtype=False)
        if t.dim() != 2 or t.shape != cos.shape or 2 * t.shape[1] > D:
            raise ValueError(f"cos and sin must both be (rows, half) with 2 * half <= {D}; got "
                             f"{tuple(cos.shape)} and {tuple(sin.shape)}")
        if t.dtype not in (torch.float32, torch.float64):
            raise TypeError(f"{name} must be float32 (or float64); got {t.dtype}")
        if t.requires_grad:
            raise ValueError(f"{name} takes no gradient")
    if positions is None:
        if L > cos.shape[0]:
            raise ValueError(f"cos and sin have {cos.shape[0]} rows for {L} tokens")
        return None
    shape = (L,) if positions.dim() == 1 else (B, L)
    return _whole("positions", positions, shape, q)


def _check_buckets(table: torch.Tensor, buckets: Optional[torch.Tensor], name: str
                   ) -> torch.Tensor:
    if table.dim() != 2 or table.shape[0] < 1:
        raise ValueError(f"{name} must be (num_buckets, heads); got {tuple(table.shape)}")
    if not table.is_floating_point():
        raise TypeError(f"{name} must be floating point; got {table.dtype}")
    if buckets is None or buckets.dim() != 1 or buckets.shape[0] % 2 == 0 \
            or buckets.shape[0] > 2 * MAX_REACH + 1:
        raise ValueError(f"buckets must be (2 * reach + 1,) with reach <= {MAX_REACH}")
    if table.shape[0] > 2 * MAX_REACH + 1:
        raise ValueError(f"{name} has more than {2 * MAX_REACH + 1} buckets")
    return _whole("buckets", buckets, buckets.shape, table)


def _check_attention(q, k, v, scale, cap, causal, prefix, documents, lengths, slopes, bias_table,
                     buckets) -> dict:
    """The checked call, as the native functions take it."""
    if not (q.dim() == k.dim() == v.dim() == 4 and q.dtype is k.dtype is v.dtype
            and q.dtype.is_floating_point and q.device == k.device == v.device):
        for name, t in (("q", q), ("k", k), ("v", v)):
            _heads(t, name)
            _same(name, t, q)
    B, Hq, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"k and v must both be ({B}, heads, tokens, {D}); got {tuple(k.shape)} "
                         f"and {tuple(v.shape)}")
    if (Hk == 0 and Hq) or (Hk and Hq % Hk):
        raise ValueError(f"the {Hq} heads of q must be a multiple of the {Hk} of k")
    if D < 1:
        raise ValueError("the head width must be at least 1")
    scale = D ** -0.5 if scale is None else float(scale)
    cap = 0.0 if cap is None else float(cap)
    if not math.isfinite(scale) or not math.isfinite(cap) or cap < 0:
        raise ValueError(f"scale and cap must be finite and cap not negative; got {scale}, {cap}")
    if prefix is not None and not causal:
        raise ValueError("prefix needs causal=True: without it every key is seen already")
    if slopes is not None:
        if tuple(slopes.shape) != (Hq,):
            raise ValueError(f"slopes must be ({Hq},); got {tuple(slopes.shape)}")
        if not slopes.is_floating_point():
            raise TypeError(f"slopes must be floating point; got {slopes.dtype}")
        _same("slopes", slopes, q, dtype=False)
        if slopes.requires_grad:
            raise ValueError("slopes take no gradient; a learned bias is bias_table's")
        slopes = slopes.to(_acc(q)).contiguous()
    if bias_table is not None:
        _same("bias_table", bias_table, q)
        buckets = _check_buckets(bias_table, buckets, "bias_table")
        if bias_table.shape[1] != Hq:
            raise ValueError(f"bias_table must have {Hq} heads; got {tuple(bias_table.shape)}")
    elif buckets is not None:
        raise ValueError("buckets come with a bias_table")
    return {"scale": scale, "cap": cap, "causal": bool(causal),
            "prefix": _whole("prefix", prefix, (B,), q),
            "documents": _documents(documents, (B, Lk), q),
            "lengths": _whole("lengths", lengths, (B,), q), "slopes": slopes,
            "bias_table": bias_table, "buckets": buckets}


# ---------------------------------------------------------------------------
# CPU reference implementations (pure PyTorch, differentiable)
# ---------------------------------------------------------------------------

def qk_norm_rotary_reference(q, k, q_weight, k_weight, cos, sin, positions=None, *,
                             eps: float = 1e-6, interleaved: bool = False
                             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """CPU reference for ``qk_norm_rotary``."""
    positions = _check_norm(q, k, q_weight, k_weight, cos, sin, positions)
    L = q.shape[2]
    at = torch.arange(L, device=q.device) if positions is None else positions.long()
    rows, half = cos.shape
    ok = ((at >= 0) & (at < rows))[..., None]
    acc = _acc(q)

    def picked(t):
        if rows == 0:
            return at.new_full((*at.shape, half), float("nan"), dtype=acc)
        return torch.where(ok, t.to(acc)[at.clamp(0, rows - 1)], float("nan"))

    c, s = picked(cos), picked(sin)
    if c.dim() == 3:
        c, s = c[:, None], s[:, None]
    out = []
    for x, w in ((q, q_weight), (k, k_weight)):
        y = x.to(acc)
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
        if w is not None:
            y = y * w.to(acc)
        turn, rest = y[..., :2 * half], y[..., 2 * half:]
        if interleaved:
            a, b = turn[..., 0::2], turn[..., 1::2]
            turn = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
        else:
            a, b = turn[..., :half], turn[..., half:]
            turn = torch.cat((a * c - b * s, a * s + b * c), -1)
        out.append(torch.cat((turn, rest), -1).to(x.dtype))
    return out[0], out[1]


def _table_rows(table: torch.Tensor, buckets: torch.Tensor) -> torch.Tensor:
    """The table's row of each relative position, NaN for a bucket it lacks."""
    b = buckets.long()
    ok = (b >= 0) & (b < table.shape[0])
    return torch.where(ok[:, None], table[b.clamp(0, table.shape[0] - 1)], float("nan"))


def relative_position_bias_reference(table: torch.Tensor, buckets: torch.Tensor, q_len: int,
                                     k_len: int) -> torch.Tensor:
    """CPU reference for ``relative_position_bias``."""
    buckets = _check_buckets(table, buckets, "table")
    reach = (buckets.numel() - 1) // 2
    at = torch.arange(q_len, device=table.device)[:, None] + (k_len - q_len)
    rel = (torch.arange(k_len, device=table.device)[None] - at).clamp(-reach, reach) + reach
    return _table_rows(table.to(_acc(table)), buckets)[rel].permute(2, 0, 1).to(table.dtype)


def _seen(rules: dict, B: int, Lq: int, Lk: int, device):
    """(relative positions, visibility), both (B, Lq, Lk)."""
    n = torch.full((B,), Lk, device=device) if rules["lengths"] is None \
        else rules["lengths"].long().clamp(0, Lk)
    j = torch.arange(Lk, device=device)
    p = torch.arange(Lq, device=device) + (n - Lq)[:, None]           # (B, Lq)
    rel = j - p[:, :, None]
    see = (j < n[:, None])[:, None, :].expand(rel.shape)
    if rules["causal"]:
        near = rel <= 0
        if rules["prefix"] is not None:
            near = near | (j < rules["prefix"].long()[:, None])[:, None, :]
        see = see & near
    if rules["documents"] is not None:
        d = rules["documents"].long()
        own = torch.gather(d, 1, p.clamp(0, max(Lk - 1, 0))) if Lk else p
        own = torch.where(p >= 0, own, -1)[:, :, None]
        see = see & (own == d[:, None, :]) & (own >= 0)
    return rel, see


def biased_attention_reference(q, k, v, *, scale: Optional[float] = None,
                               cap: Optional[float] = None, causal: bool = False, prefix=None,
                               documents=None, lengths=None, slopes=None, bias_table=None,
                               buckets=None, return_log_degree: bool = False):
    """CPU reference for ``biased_attention``."""
    r = _check_attention(q, k, v, scale, cap, causal, prefix, documents, lengths, slopes,
                         bias_table, buckets)
    acc = _acc(q)
    B, Hq, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    per = Hq // Hk if Hk else 1
    rel, see = _seen(r, B, Lq, Lk, q.device)
    see = see[:, None]
    # what no query sees, whatever it holds, is out of every product
    dead = ~see.any(2)[:, :, :, None]
    kd, vd = (torch.where(dead, 0.0, t.to(acc)).repeat_interleave(per, 1) for t in (k, v))
    s = torch.matmul(q.to(acc), kd.transpose(2, 3).contiguous()) * r["scale"]
    if r["cap"]:
        s = r["cap"] * torch.tanh(s / r["cap"])
    if r["slopes"] is not None:
        s = s - r["slopes"][:, None, None] * rel.abs()[:, None]
    if bias_table is not None:
        reach = (r["buckets"].numel() - 1) // 2
        rows = _table_rows(bias_table.to(acc), r["buckets"])
        s = s + rows[rel.clamp(-reach, reach) + reach].permute(0, 3, 1, 2)
    s = torch.where(see, s, _NEG_INF)
    m = s.detach().amax(-1, keepdim=True) if Lk else s.new_full((B, Hq, Lq, 1), _NEG_INF)
    m = torch.where(m == _NEG_INF, 0.0, m)
    e = torch.where(see, torch.exp(s - m), 0.0)
    z = e.sum(-1, keepdim=True)
    empty = z == 0
    out = torch.where(empty, 0.0, torch.matmul(e, vd) / torch.where(empty, 1.0, z)).to(q.dtype)
    if not return_log_degree:
        return out
    log_C = torch.where(empty, _NEG_INF, m + torch.log(torch.where(empty, 1.0, z)))
    return out, log_C.squeeze(-1)


# ---------------------------------------------------------------------------
# Calls under torch.jit.trace
# ---------------------------------------------------------------------------

class _TracedCall(torch.autograd.Function):
    """A call as one step of a trace, which records a Python function as what is to
    be run again, but nothing of what C++ does with the tensors' memory."""

    @staticmethod
    def forward(ctx, call, *tensors):
        ctx.set_materialize_grads(False)
        with torch.enable_grad():
            ctx.leaves = [t if t is None else t.detach().requires_grad_(t.requires_grad)
                          for t in tensors]
            out = call(*ctx.leaves)
        ctx.out = out if isinstance(out, tuple) else (out,)
        out = tuple(t.detach() for t in ctx.out)
        return out if len(out) > 1 else out[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *upstream):
        want = [n for n, t in enumerate(ctx.leaves) if t is not None and t.requires_grad]
        outs = [(t, g) for t, g in zip(ctx.out, upstream) if g is not None]
        got = torch.autograd.grad([t for t, _ in outs], [ctx.leaves[n] for n in want],
                                  [g for _, g in outs], retain_graph=True, allow_unused=True)
        grads = [None] * len(ctx.leaves)
        for n, g in zip(want, got):
            grads[n] = g
        return (None, *grads)


def _traceable(call, tensors, **rules):
    # (the kernels read memory, which holds a conjugate's imaginary part with the other sign)
    tensors = [t.resolve_neg() if isinstance(t, torch.Tensor) and t.is_neg() else t for t in tensors]
    if not torch.jit.is_tracing():
        return call(*tensors, **rules)
    return _TracedCall.apply(functools.partial(call, **rules), *tensors)


# ---------------------------------------------------------------------------
# Public API
# ---------------------------------------------------------------------------

def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, q_weight: Optional[torch.Tensor],
                   k_weight: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor,
                   positions: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                   interleaved: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """Norm of queries and keys for each head, then the rotation by position.

        y = x / sqrt(mean(x^2) + eps) * weight
        (a, b) -> (a cos - b sin, a sin + b cos)

    q (B, Hq, L, D) and k (B, Hk, L, D) of any strides (a projection's
    (B, L, H, D) transposed is read where it lies); weights (D,) in their type
    or None.  cos, sin (rows, half), float32, from ``rotary_table``: the first
    2 * half of the D elements turn in pairs (i, i + half), or (2i, 2i + 1) with
    `interleaved`, the others are left as normed.  `positions`: the row of each
    token, integers (L,) or (B, L); None takes 0 .. L-1.  A position outside
    the table makes its tokens NaN.  D <= 512 on the GPU.

    Returns contiguous (q', k') in the inputs' type.  Differentiable in q, k and
    the weights; the weights' gradients are summed in a fixed order."""
    if not q.is_cuda:
        return qk_norm_rotary_reference(q, k, q_weight, k_weight, cos, sin, positions, eps=eps,
                                        interleaved=interleaved)
    done = _C and _C.norm_rotary_as_is(q, k, q_weight, k_weight, cos, sin, positions, eps,
                                       interleaved)
    if done is not None:
        return done
    return _traceable(_norm_rotary, (q, k, q_weight, k_weight, cos, sin, positions), eps=eps,
                      interleaved=interleaved)


def _norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, *, eps, interleaved):
    positions = _check_norm(q, k, q_weight, k_weight, cos, sin, positions)
    if q.shape[3] > 512:
        raise ValueError(f"heads wider than 512 are not served on the GPU; got {q.shape[3]}")
    ops._require_cuda_ext("qk_norm_rotary")
    w = [None if t is None else t.contiguous() for t in (q_weight, k_weight)]
    return _C.norm_rotary(q, k, w[0], w[1], cos.float().contiguous(), sin.float().contiguous(),
                          positions, eps, interleaved)


def relative_position_bias(table: torch.Tensor, buckets: torch.Tensor, q_len: int, k_len: int
                           ) -> torch.Tensor:
    """The learned bias of every query and key, (H, q_len, k_len):

        out[h, i, j] = table[buckets[clamp(j - (i + k_len - q_len))], h]

    table (num_buckets, H); buckets (2 * reach + 1,) integers from
    ``relative_buckets`` or of the caller's own (a bucket that the table lacks
    gives NaN).  The relative position is clamped to +-reach.  Differentiable in
    the table; its gradient is summed in fp32 in a fixed order.
    ``biased_attention`` takes table and buckets themselves, without this tensor."""
    if q_len < 0 or k_len < 0:
        raise ValueError(f"q_len and k_len must not be negative; got {q_len}, {k_len}")
    if not table.is_cuda:
        return relative_position_bias_reference(table, buckets, q_len, k_len)
    done = _C and _C.position_bias_as_is(table, buckets, q_len, k_len)
    if done is not None:
        return done
    return _traceable(_position_bias, (table, buckets), q_len=q_len, k_len=k_len)


def _position_bias(table, buckets, *, q_len, k_len):
    buckets = _check_buckets(table, buckets, "table")
    ops._require_cuda_ext("relative_position_bias")
    return _C.position_bias(table, buckets, q_len, k_len)


def biased_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *,
                     scale: Optional[float] = None, cap: Optional[float] = None,
                     causal: bool = False, prefix: Optional[torch.Tensor] = None,
                     documents: Optional[torch.Tensor] = None,
                     lengths: Optional[torch.Tensor] = None,
                     slopes: Optional[torch.Tensor] = None,
                     bias_table: Optional[torch.Tensor] = None,
                     buckets: Optional[torch.Tensor] = None, return_log_degree: bool = False):
    """Attention with capped scores, distance biases and masks:

        x = scale * q_i . k_j        s = cap * tanh(x / cap)       (no cap: s = x)
        s = s - slopes[h] * |j - p| + bias_table[buckets[clamp(j - p)], h]
        D_i = sum_j exp(s) v_j / sum_j exp(s)        log_C_i = log sum_j exp(s)

    over the keys that query i, at position p, sees.  q (B, Hq, Lq, D), k and v
    (B, Hk, Lk, D), Hq a multiple of Hk (query head h reads key head
    h // (Hq // Hk)); scale defaults to D ** -0.5.

    * lengths (B,): only the first lengths[b] keys are filled (a cache); the
      queries are the last Lq of them, p = i + lengths[b] - Lq.
    * causal: keys after p are not seen, except the first prefix[b] ones, which
      every query sees.
    * documents (B, Lk): several sequences in one row; a query sees the keys of
      its own position's document only, and a negative one (padding) sees nothing
      and is not seen.  Any integers: int32 is taken as it is, 64-bit numbers are
      written anew as int32 in every call (one small launch).
    * slopes (Hq,): linear distance bias, no gradient.
    * bias_table (num_buckets, Hq) with buckets (2 * reach + 1,): a learned bias
      by buckets of the relative position, as ``relative_position_bias`` writes
      out; it has q's type and its gradient is summed in fp32.  -inf in it
      excludes the distance.

    A row that sees nothing gives 0 (and log_C = -inf).  What a query does not
    see adds nothing to it, whatever it holds.

    Returns D in q's type (and with q's order of heads and tokens in memory), or
    (D, log_C) with return_log_degree, log_C fp32 (B, Hq, Lq).  Differentiable in
    q, k, v and bias_table; the gradients are summed in a fixed order.  The GPU
    serves fp16, bf16 and fp32 with D <= 128 (a width that is no multiple of 8,
    or rows that do not start on 16 bytes, are copied first), a scale within fp32 and
    caps of 2^-60 to 2^60."""
    if not q.is_cuda:
        return biased_attention_reference(
            q, k, v, scale=scale, cap=cap, causal=causal, prefix=prefix, documents=documents,
            lengths=lengths, slopes=slopes, bias_table=bias_table, buckets=buckets,
            return_log_degree=return_log_degree)
    done = _C and _C.attention_as_is(q, k, v, scale, cap, causal, prefix, documents, lengths,
                                     slopes, bias_table, buckets, return_log_degree)
    if done is not None:
        return done if return_log_degree else done[0]
    return _traceable(_attention, (q, k, v, prefix, documents, lengths, slopes, bias_table, buckets),
                      scale=scale, cap=cap, causal=causal, return_log_degree=return_log_degree)


def _attention(q, k, v, prefix, documents, lengths, slopes, bias_table, buckets, *, scale, cap,
               causal, return_log_degree):
    rules = _check_attention(q, k, v, scale, cap, causal, prefix, documents, lengths, slopes,
                             bias_table, buckets)
    D = q.shape[3]
    if D > 128:
        raise ValueError(f"heads wider than 128 are not served on the GPU; got {D}")
    ops._require_cuda_ext("biased_attention")
    docs = rules["documents"]
    if docs is not None and docs.dtype is not torch.int32:
        docs = _C.document_ids(docs)
    if D % 8:
        q, k, v = (torch.nn.functional.pad(t, (0, -D % 8)) for t in (q, k, v))
    out, log_C = _C.attention(q, k, v, rules["bias_table"], rules["lengths"], rules["prefix"],
                              docs, rules["slopes"], rules["buckets"],
                              rules["scale"], rules["cap"], rules["causal"], return_log_degree)
    if D % 8:
        out = out[..., :D]
    return (out, log_C) if return_log_degree else out


__all__ = [
    "qk_norm_rotary",
    "relative_position_bias",
    "biased_attention",
    "rotary_table",
    "relative_buckets",
    "qk_norm_rotary_reference",
    "relative_position_bias_reference",
    "biased_attention_reference",
]

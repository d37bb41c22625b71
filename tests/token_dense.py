"""biased_attention's values and gradients in 64 bits as dense tensors on the
inputs' device, for sizes at which the pair by pair oracle takes seconds."""
from __future__ import annotations

import torch


def seen(B, Lq, Lk, device, causal=False, documents=None, lengths=None):
    """(relative positions, visibility), both (B, Lq, Lk)."""
    n = torch.full((B,), Lk, device=device) if lengths is None else lengths.long().clamp(0, Lk)
    j, p = torch.arange(Lk, device=device), torch.arange(Lq, device=device) + (n - Lq)[:, None]
    rel = j - p[:, :, None]
    see = (j < n[:, None])[:, None, :].expand(rel.shape)
    if causal:
        see = see & (rel <= 0)
    if documents is not None:
        own = torch.where(p >= 0, documents.long().gather(1, p.clamp(0)), -1)[:, :, None]
        see = see & (own == documents[:, None, :]) & (own >= 0)
    return rel, see


def attention(q, k, v, go, *, scale=None, cap=None, causal=False, documents=None, lengths=None,
              bias_table=None, buckets=None):
    """{out, gq, gk, gv} in 64 bits."""
    B, Hq, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    per = Hq // Hk
    rel, see = seen(B, Lq, Lk, q.device, causal, documents, lengths)
    leaves = [t.detach().double().requires_grad_() for t in (q, k, v)]
    Q, K, V = leaves[0], *(t.repeat_interleave(per, 1) for t in leaves[1:])
    s = torch.matmul(Q, K.transpose(2, 3).contiguous()) * (D ** -0.5 if scale is None else scale)
    if cap:
        s = cap * torch.tanh(s / cap)
    if bias_table is not None:
        R = (len(buckets) - 1) // 2
        s = s + bias_table.double()[buckets.long()[rel.clamp(-R, R) + R]].permute(0, 3, 1, 2)
    s = s.masked_fill(~see[:, None], -float("inf"))
    top = s.detach().amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top.isinf(), 0.0, top))
    z = e.sum(-1, keepdim=True)
    out = torch.matmul(e, V) / torch.where(z == 0, 1.0, z)
    grads = torch.autograd.grad(out, leaves, go.double())
    return {"out": out.detach(), **dict(zip(("gq", "gk", "gv"), grads))}

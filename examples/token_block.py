"""The token operators together: a small attention block, trained on packed
documents and then run token by token over a cache.

    python examples/token_block.py [--device cuda] [--steps 60]

Queries and keys are normed per head and rotated by position
(``qk_norm_rotary``); the attention (``biased_attention``) caps its scores, adds
a learned bias by buckets of the distance, keeps documents apart in training and
reads a cache of mixed lengths in decoding.  What the bias has learned is read off
it written out (``relative_position_bias``).  The task is to repeat the token that
stood `lag` places earlier in the same document.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn
from torch.nn import functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from neural_shift_cuda import (biased_attention, qk_norm_rotary, relative_buckets,  # noqa: E402
                               relative_position_bias, rotary_table)


class TokenBlock(nn.Module):
    def __init__(self, vocab=32, heads=4, key_heads=2, width=32, cap=30.0, buckets=16, reach=48,
                 longest=512, device=None, dtype=torch.float32):
        super().__init__()
        self.heads, self.key_heads, self.width, self.cap = heads, key_heads, width, cap
        dim, kw = heads * width, {"device": device, "dtype": dtype}
        self.embed = nn.Embedding(vocab, dim, **kw)
        self.qkv = nn.Linear(dim, (heads + 2 * key_heads) * width, bias=False, **kw)
        self.out = nn.Linear(dim, vocab, **kw)
        self.q_weight = nn.Parameter(torch.ones(width, **kw))
        self.k_weight = nn.Parameter(torch.ones(width, **kw))
        self.bias = nn.Parameter(torch.zeros(buckets, heads, **kw))
        cos, sin = rotary_table(longest, width, device=device)
        self.register_buffer("cos", cos)
        self.register_buffer("sin", sin)
        self.register_buffer("buckets", relative_buckets(buckets, reach, bidirectional=False,
                                                         device=device))

    def qkv_of(self, tokens, positions):
        """q, k, v (B, heads, T, width): normed, and turned to their positions."""
        B, T = tokens.shape
        x = self.qkv(self.embed(tokens)).view(B, T, -1, self.width).transpose(1, 2)
        q, k, v = x.split([self.heads, self.key_heads, self.key_heads], 1)
        q, k = qk_norm_rotary(q, k, self.q_weight, self.k_weight, self.cos, self.sin, positions)
        return q, k, v

    def attend(self, q, k, v, **masks):
        y = biased_attention(q, k, v, cap=self.cap, causal=True, bias_table=self.bias,
                             buckets=self.buckets, **masks)
        return self.out(y.transpose(1, 2).flatten(2))

    @torch.no_grad()
    def bias_by_distance(self, reach):
        """(heads, reach + 1): the bias of a key 0, 1, .. reach places back."""
        return relative_position_bias(self.bias, self.buckets, 1, reach + 1)[:, 0].flip(1)

    def forward(self, tokens, documents=None):
        positions = torch.arange(tokens.shape[1], device=tokens.device)
        return self.attend(*self.qkv_of(tokens, positions), documents=documents)


class Cache:
    """Keys and values of sequences at lengths of their own."""

    def __init__(self, block: TokenBlock, batch: int, longest: int):
        w = block.qkv.weight
        self.k, self.v = (torch.empty(batch, block.key_heads, longest, block.width,
                                      device=w.device, dtype=w.dtype) for _ in range(2))
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=w.device)

    @torch.no_grad()
    def step(self, block: TokenBlock, tokens):
        """Logits (B, vocab) after one more token for every sequence."""
        q, k, v = block.qkv_of(tokens[:, None], self.lengths[:, None])
        rows = torch.arange(tokens.shape[0], device=tokens.device)
        at = self.lengths.long()
        self.k[rows, :, at], self.v[rows, :, at] = k[:, :, 0], v[:, :, 0]
        self.lengths += 1
        return block.attend(q, self.k, self.v, lengths=self.lengths)[:, 0]


def batch_of(gen, B, T, vocab, lag, device):
    """Tokens, documents packed into the rows, and where a target exists."""
    tokens = torch.randint(1, vocab, (B, T), generator=gen)
    documents = torch.zeros(B, T, dtype=torch.int32)
    starts = torch.zeros(B, T, dtype=torch.int64)
    for b in range(B):
        for n, c in enumerate(sorted(torch.randint(2, T - 1, (3,), generator=gen).tolist())):
            documents[b, c:], starts[b, c:] = n + 1, c
    target = torch.roll(tokens, lag, 1)
    known = torch.arange(T)[None] - starts >= lag
    return tokens.to(device), documents.to(device), target.to(device), known.to(device)


def main(argv=None) -> float:
    ap = argparse.ArgumentParser()
    ap.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--tokens", type=int, default=160)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    gen = torch.Generator().manual_seed(1)
    block = TokenBlock(device=a.device)
    opt = torch.optim.Adam(block.parameters(), 3e-3)
    for step in range(a.steps):
        tokens, documents, target, known = batch_of(gen, 8, a.tokens, 32, 3, a.device)
        loss = F.cross_entropy(block(tokens, documents)[known], target[known])
        opt.zero_grad()
        loss.backward()
        opt.step()
        if step % 10 == 0 or step + 1 == a.steps:
            print(f"step {step:3d}  loss {loss.item():.4f}", flush=True)
    bias = block.bias_by_distance(8).float().cpu()
    print("learned bias by distance, mean of the heads: "
          + " ".join(f"{b:+.3f}" for b in bias.mean(0).tolist()))
    # token by token gives what the whole sequence gives
    tokens = batch_of(gen, 4, 24, 32, 3, a.device)[0]
    cache = Cache(block, 4, 64)
    with torch.no_grad():
        whole = block(tokens)
        one = torch.stack([cache.step(block, tokens[:, t]) for t in range(tokens.shape[1])], 1)
    off = float((one - whole).abs().max())
    print(f"one token at a time: largest difference from the whole sequence {off:.2e}")
    return off


if __name__ == "__main__":
    main()

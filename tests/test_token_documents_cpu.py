"""Document numbers, positions and lengths of every integer type and size: which
documents are one, and values beyond int32 at its ends."""
from __future__ import annotations

import pytest
import torch

from neural_shift_cuda import biased_attention, qk_norm_rotary, rotary_table

TOP = 1 << 31

# (type, numbers); each is the packing 0 0 0 1 1 0 2 - - 1 of a row of ten
PACKINGS = {
    "int32": (torch.int32, (7, 9, 1)),
    "int64": (torch.int64, (TOP, TOP + 1, 5)),
    "int64, far apart": (torch.int64, ((1 << 63) - 1, 3, 1 << 62)),
    "int64, equal in their lower halves": (torch.int64, (4, 4 + (1 << 32), 4 + (1 << 33))),
    "uint32": (torch.uint32, (TOP + 1, (1 << 32) - 1, 3)),
    "uint64": (torch.uint64, ((1 << 64) - 1, 1 << 63, 12)),
    "int16": (torch.int16, (300, 2, 1)),
    "uint8": (torch.uint8, (200, 255, 0)),
}
ORDER = (0, 0, 0, 1, 1, 0, 2, None, None, 1)
SIGNED = (torch.int32, torch.int64, torch.int16)


def packed(dtype, numbers):
    """Documents of two rows, and the same as small numbers."""
    pad = -5 if dtype in SIGNED else None
    row = [numbers[n] if n is not None else pad for n in ORDER]
    small = [n if n is not None else -1 for n in ORDER]
    if pad is None:  # without padding: those places belong to the last number
        row = [numbers[2] if x is None else x for x in row]
        small = [2 if n < 0 else n for n in small]
    rows, smalls = [row, row[::-1]], [small, small[::-1]]
    if dtype in (torch.uint32, torch.uint64):  # torch makes these from the signed type's bits
        bits = 32 if dtype is torch.uint32 else 64
        wide = [[x - (1 << bits) if x >> (bits - 1) else x for x in r] for r in rows]
        t = torch.tensor(wide, dtype=torch.int32 if bits == 32 else torch.int64).view(dtype)
    else:
        t = torch.tensor(rows, dtype=dtype)
    return t, torch.tensor(smalls, dtype=torch.int32)


def tensors(dtype=torch.float32):
    g = torch.Generator().manual_seed(4)
    return [torch.randn(2, 2, 10, 8, generator=g, dtype=dtype) for _ in range(3)]


@pytest.mark.parametrize("name", list(PACKINGS))
@pytest.mark.parametrize("causal", [False, True])
def test_documents_are_told_apart(name, causal):
    docs, small = packed(*PACKINGS[name])
    q, k, v = tensors()
    got = biased_attention(q, k, v, causal=causal, documents=docs)
    assert torch.equal(got, biased_attention(q, k, v, causal=causal, documents=small))
    assert not torch.equal(got, biased_attention(q, k, v, causal=causal))


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32, torch.uint64])
@pytest.mark.parametrize("n", [4, 10, (1 << 32) + 4, (1 << 63) + 4])
def test_lengths_beyond_int32_are_whole(dtype, n):
    if n >= 1 << 63 and dtype is not torch.uint64 or n >= 1 << 32 and dtype is torch.uint32:
        pytest.skip("beyond the type")
    bits = n - (1 << 64) if n >> 63 else n
    lengths = torch.tensor([bits, 3], dtype=torch.int64)
    lengths = lengths.view(dtype) if dtype is torch.uint64 else lengths.to(dtype)
    q, k, v = tensors()
    want = biased_attention(q, k, v, lengths=torch.tensor([min(n, 10), 3], dtype=torch.int32))
    assert torch.equal(biased_attention(q, k, v, lengths=lengths), want)


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32, torch.uint64])
def test_positions_beyond_int32_are_outside(dtype):
    q, k, _ = tensors()
    cos, sin = rotary_table(20, 8)
    at = torch.arange(10)
    at[3] = (1 << 32) + 2 if dtype is not torch.uint32 else (1 << 31) + 2
    out = qk_norm_rotary(q, k, None, None, cos, sin, at.to(dtype))[0]
    assert out[:, :, 3].isnan().all() and not out[:, :, 4].isnan().any()

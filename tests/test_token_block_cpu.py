"""The example of the token operators on the CPU, and the native entries'
refusal of token strides beyond their 32-bit offsets."""
from __future__ import annotations

import ctypes
import importlib.util
import os

import pytest
import torch

from test_token_ops_cpu import attention_args, native


def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                        "token_block.py")
    spec = importlib.util.spec_from_file_location("token_block", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_token_block_learns_and_decodes():
    # the logits' sums of 128 products of unit size and the few steps behind them
    assert example().main(["--device", "cpu", "--steps", "3", "--tokens", "40"]) < 1e-4


def test_decoding_with_mixed_lengths():
    m = example()
    torch.manual_seed(0)
    block = m.TokenBlock().double()
    cache = m.Cache(block, 2, 16)
    tokens = torch.randint(1, 32, (2, 6))
    for t in range(3):
        cache.step(block, tokens[:, t])
    cache.lengths[1] = 1  # the second sequence goes back to its first token
    got = cache.step(block, torch.stack((tokens[0, 3], tokens[1, 1])))
    with torch.no_grad():
        for b, n in ((0, 4), (1, 2)):
            want = block(tokens[b:b + 1, :n])[0, -1]
            assert float((got[b] - want).abs().max()) < 1e-6  # float32 tables of the angles


@pytest.mark.parametrize("over", [{"q_stride": (64, 32, 1 << 23)}, {"k_stride": (32, 32, 1 << 23)},
                                  {"v_stride": (32, 32, -8)}])
def test_token_strides_served(over):
    C = native()
    with pytest.raises(RuntimeError, match="token strides"):
        C._call("nsh_attention_forward", ctypes.byref(attention_args(**{"dtype": 3, **over})), None)

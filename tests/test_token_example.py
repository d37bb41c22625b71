"""The token block's learned bias, read off written out, is the table's."""
from __future__ import annotations

import torch

from test_token_block_cpu import example


def test_bias_by_distance_is_the_tables():
    block = example().TokenBlock(heads=3, key_heads=1, buckets=8, reach=20)
    with torch.no_grad():
        block.bias.normal_(generator=torch.Generator().manual_seed(0))
    got = block.bias_by_distance(25)
    ids = block.buckets[20 - torch.arange(26).clamp(max=20)]  # keys before the query
    assert torch.equal(got, block.bias.detach()[ids.long()].t())


def test_the_example_runs_the_three_operators_together(capsys):
    example().main(["--device", "cpu", "--steps", "2", "--tokens", "30"])
    out = capsys.readouterr().out
    assert "learned bias by distance" in out and "one token at a time" in out

"""The position bias's gradient over so many rows that a turn of its workgroups
is 2^32 places and more."""
from __future__ import annotations

import pytest
import torch

from neural_shift_cuda import relative_position_bias

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


@pytest.mark.parametrize("rows", [(1 << 25) - 17, 1 << 25, (1 << 25) + 16 * 5 + 3])
@pytest.mark.parametrize("k_len", [1, 3])
def test_gradient_of_many_rows(rows, k_len):
    """Upstream values of 0 and 1 in one place of sixteen: every sum is a whole
    number below 2^24, and exact."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    go = (torch.rand(1, rows, k_len, generator=g, device="cuda") < 1 / 16).float()
    buckets = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    table = torch.zeros(3, 1, device="cuda", requires_grad=True)
    (got,) = torch.autograd.grad(relative_position_bias(table, buckets, rows, k_len), table, go)
    at = torch.arange(k_len, device="cuda")[None] - (torch.arange(rows, device="cuda")[:, None]
                                                     + k_len - rows)
    ids = buckets.long()[at.clamp(-1, 1) + 1]
    want = [int(go[0][ids == b].double().sum()) for b in range(3)]
    assert sum(want) < 1 << 24 and got[:, 0].tolist() == want

"""Gradients by keys where a key block's queries are shared by more workgroups
than it has tiles of them: single heads, causal, whose last keys are seen by few
rows."""
from __future__ import annotations

import pytest
import torch

from test_gpu_attention import check, inputs

pytestmark = [
    pytest.mark.gpu,
    pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU"),
]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [96, 128])
@pytest.mark.parametrize("cap", [None, 20.0])
def test_parts_without_rows(dtype, D, cap):
    q, k, v, go, _ = inputs(1, 1, 1, 1024, 1024, D, dtype)
    check(q, k, v, go, {"causal": True, "cap": cap})


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_parts_without_rows_of_a_short_cache(dtype):
    q, k, v, go, _ = inputs(2, 2, 1, 700, 900, 128, dtype)
    check(q, k, v, go, {"causal": True, "lengths": torch.tensor([900, 130], dtype=torch.int32)})

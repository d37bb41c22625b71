"""Scales and caps that fp32 does not hold are refused by the native entry: a cap
below its smallest number would be none, one beyond its largest gives no number."""
from __future__ import annotations

import ctypes

import pytest

from test_token_ops_cpu import attention_args, native


@pytest.mark.parametrize("over", [{"cap": 1e-46}, {"cap": 1e-40}, {"cap": 1e39}, {"cap": 1e30},
                                  {"scale": 1e39}, {"scale": -1e300}])
def test_beyond_fp32(over):
    C = native()
    with pytest.raises(RuntimeError, match="within fp32"):
        C._call("nsh_attention_forward", ctypes.byref(attention_args(**{"dtype": 3, **over})), None)

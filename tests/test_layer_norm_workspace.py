"""layer_norm's scratch memory for the weights' gradients: as large as what the launches
write, and small next to the rows."""
from __future__ import annotations

import ctypes

import pytest
import torch

from neural_shift_cuda_amd import _C

CODES = {torch.float16: 1, torch.bfloat16: 2, torch.float32: 3}


def size(rows, n, dtype):
    a = _C._LayerNormArgs(rows=rows, n=n, dtype=CODES[dtype])
    return _C._lib.nsh_layer_norm_workspace_bytes(ctypes.byref(a))


@pytest.mark.parametrize("rows,n,dtype", [(512, 1000000, torch.float32), (2000, 100000, torch.bfloat16),
                                          (600, 40000, torch.bfloat16), (70000, 16392, torch.float16)])
def test_wide_rows(rows, n, dtype):
    """Sets of two sums a column: 16 waves a CU have 64 x 16 bytes of columns each, and one set
    there is in any case."""
    sums = 16 * 256 * 64 * (16 // dtype.itemsize)
    got = size(rows, n, dtype)
    assert got % (8 * n) == 0 and 8 * n <= got <= 8 * (sums + 2 * n)
    assert got < rows * n * dtype.itemsize / 2


def test_rows_of_512_lanes():
    """One workgroup a CU, of which there are 256."""
    assert size(3000, 16384, torch.float16) == 256 * 2 * 16384 * 4
    assert size(40, 16384, torch.float16) == 40 * 2 * 16384 * 4


def test_no_size_without_a_type():
    a = _C._LayerNormArgs(rows=4, n=8)
    assert _C._lib.nsh_layer_norm_workspace_bytes(ctypes.byref(a)) == -1


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")
@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("n", [8, 60, 250, 500, 1000, 2000, 4000, 8000, 16000, 20000, 70000])
def test_the_launches_stay_inside(n, dtype):
    """Every form of a row: what lies behind the workspace is left as it was, every sum in it is
    written, and one byte less is refused."""
    for rows in (3, 300, 1100):
        g = torch.Generator(device="cuda").manual_seed(n + rows)
        x, gy = (torch.randn(rows, n, generator=g, device="cuda").to(dtype) for _ in range(2))
        stats = torch.stack((x.float().mean(-1), (x.float().var(-1, correction=0) + 1e-5) ** -0.5), 1).contiguous()
        need, room = size(rows, n, dtype), 1 << 16
        ws = torch.full((need + room,), 0xA5, dtype=torch.uint8, device="cuda")
        gw, gb = torch.empty(2, n, dtype=dtype, device="cuda")
        a = _C._LayerNormArgs(x=x.data_ptr(), rows=rows, n=n, x_stride=n, eps=1e-5, dtype=CODES[dtype],
                              stats=stats.data_ptr(), grad_y=gy.data_ptr(), gy_stride=n, grad_weight=gw.data_ptr(),
                              grad_bias=gb.data_ptr(), workspace=ws.data_ptr(), workspace_bytes=need - 1)
        with pytest.raises(RuntimeError, match="workspace"):
            _C._call("nsh_layer_norm_backward", ctypes.byref(a), torch.cuda.current_stream().cuda_stream)
        a.workspace_bytes = need
        _C._call("nsh_layer_norm_backward", ctypes.byref(a), torch.cuda.current_stream().cuda_stream)
        assert (ws[need:] == 0xA5).all()
        assert not (ws[:need].view(torch.int32) == -0x5A5A5A5B).any()
        want = gy.double().sum(0)
        # a chain of at most all rows, and the result's rounding
        tol = (rows + 8) * 2.0 ** -24 * gy.double().abs().sum(0) + torch.finfo(dtype).eps / 2 * want.abs()
        assert ((gb.double() - want).abs() <= tol + 2.0 ** -24).all()

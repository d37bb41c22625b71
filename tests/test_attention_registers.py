"""The attention kernels keep everything in registers: no vector register is
spilled, and where the compiler sets memory aside (scalars that it then keeps in
vector lanes) no instruction touches it."""
from __future__ import annotations

import os
import subprocess

import pytest

from neural_shift_cuda_amd import _C, build
from test_kernel_registers import _kernels
from test_matrix_results import functions

pytestmark = pytest.mark.skipif(not os.path.exists(_C.LIBRARY_PATH), reason="library not built")


def attention_kernels():
    found = {n: k for n, k in _kernels().items() if "att_" in n}
    assert len(found) > 100
    return found


def source_of(name):
    side = "bwd" if "att_bwd" in name else "fwd"
    return f"attention_{side}_{'bf16' if 'bf16' in name else 'f16' if 'DF16_' in name else 'f32'}.hip"


def test_no_vector_register_is_spilled():
    assert not [n for n, k in attention_kernels().items() if k[".vgpr_spill_count"]]


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
def test_no_kernel_touches_scratch(tmp_path):
    left = [n for n, k in attention_kernels().items() if k[".private_segment_fixed_size"]]
    for src in sorted({source_of(n) for n in left}):
        out = tmp_path / (src + ".s")
        subprocess.run([build._hipcc(), *build._flags("test"), "-x", "hip", "--cuda-device-only",
                        "-S", os.path.join(build.CSRC, src), "-o", str(out)], check=True,
                       capture_output=True)
        code = functions(out.read_text())
        for n in left:
            if source_of(n) == src:
                assert not [s for s in code[n] if s.startswith(("scratch_", "buffer_store", "flat_"))
                            and "lds" not in s], n

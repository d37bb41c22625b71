"""No kernel of the gated projections reads or overwrites a matrix product's result before
the hardware has it, and none of theirs or of layer norm's spills or keeps an array in
memory."""
from __future__ import annotations

import concurrent.futures as cf
import os
import re
import subprocess

import pytest

from neural_shift_cuda_amd import _C, build
from test_kernel_registers import _kernels
from test_matrix_results import early, functions

SOURCES = ["gated_bf16.hip", "gated_f16.hip", "gated_f32.hip", "gated_f32_parts.hip"]


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
def test_gated_kernels(tmp_path):
    def assembly(src):
        out = tmp_path / (src + ".s")
        subprocess.run([build._hipcc(), *build._flags("test"), "-x", "hip", "--cuda-device-only",
                        "-S", os.path.join(build.CSRC, src), "-o", str(out)], check=True,
                       capture_output=True)
        return out.read_text()

    kernels = 0
    with cf.ThreadPoolExecutor(4) as ex:
        for src, text in zip(SOURCES, ex.map(assembly, SOURCES)):
            for name, code in functions(text).items():
                kernels += 1
                found = early(code)
                assert not found, f"{src}: {name}: {found[:3]}"
    assert kernels > 20


@pytest.mark.skipif(not os.path.exists(_C.LIBRARY_PATH), reason="library not built")
def test_no_spills():
    kernels = {n: k for n, k in _kernels().items() if re.search(r"(gated|layer_norm)_\w+_kernel", n)}
    assert len(kernels) > 100
    bad = {n: (k[".vgpr_spill_count"], k[".private_segment_fixed_size"]) for n, k in kernels.items()
           if k[".vgpr_spill_count"] or k[".private_segment_fixed_size"]}
    assert not bad

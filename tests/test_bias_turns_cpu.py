"""The turns in which the position bias's gradient shares its reads out: every
place once, and an end to every workgroup's walk, whatever their number."""
from __future__ import annotations

import os
import subprocess

import pytest

from neural_shift_cuda_amd import build

PROGRAM = r"""
#include <cstdio>
#include <vector>
#include "positionbias.hpp"
// every run of `whole` places is begun once; a walk may take `most` steps
static bool covered(uint32_t blocks, uint32_t run, uint32_t whole) {
    const uint64_t runs = (uint64_t(whole) + run - 1) / run, most = runs / blocks + 2;
    std::vector<unsigned char> begun(runs, 0);
    for (uint32_t block = 0; block < blocks; ++block) {
        uint64_t steps = 0;
        for (nsh::Turns t = nsh::Turns::of(block, blocks, run); t.at < whole; t.at += t.step) {
            if (t.at % run || begun[t.at / run]++ || ++steps > most) return false;
        }
    }
    for (unsigned char n : begun)
        if (n != 1) return false;
    return true;
}
int main() {
    const uint32_t blocks[] = {1, 3, 128, (1u << 21) - 1, 1u << 21, (1u << 21) + 1, 3u << 20, 1u << 24};
    const uint32_t whole[] = {0, 1, 2047, 2048, 2049, 100001, 1u << 22, (1u << 28) - 3, 1u << 28};
    for (uint32_t b : blocks)
        for (uint32_t w : whole)
            if (!covered(b, 2048, w)) {
                std::printf("%u workgroups, %u places", b, w);
                return 1;
            }
    return 0;
}
"""


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
def test_every_place_once(tmp_path):
    src, exe = tmp_path / "turns.cpp", tmp_path / "turns"
    src.write_text(PROGRAM)
    subprocess.run([build._hipcc(), *build._flags("test"), "-x", "hip", "--offload-host-only",
                    str(src), "-o", str(exe)], check=True, capture_output=True)
    ran = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert ran.returncode == 0, ran.stdout

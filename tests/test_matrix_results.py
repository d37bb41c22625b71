"""No attention kernel reads or overwrites a matrix product's result before the
hardware has it.

The results may be touched 12 wait states after a 16-bit 32 x 32 product (18
after an fp32 one) at the earliest, on every path; the hardware does not wait,
and the compiler's count has been seen to miss a copy behind a loop's exit.  The
assembly of the attention kernels, made here from source, is followed block by
block."""
from __future__ import annotations

import concurrent.futures as cf
import os
import re
import subprocess

import pytest

from neural_shift_cuda_amd import build

SOURCES = [f"attention_{d}_{t}.hip" for d in ("fwd", "bwd") for t in ("bf16", "f16", "f32")]
VGPR = re.compile(r"\bv\[(\d+):(\d+)\]|\bv(\d+)\b")


def registers(operand):
    out = []
    for lo, hi, one in VGPR.findall(operand):
        out += [int(one)] if one else range(int(lo), int(hi) + 1)
    return out


def functions(text):
    """{name: instructions and labels} of an assembly file."""
    out, cur = {}, None
    for line in text.splitlines():
        m = re.match(r"^(_Z\w+):", line)
        if m:
            cur = out.setdefault(m.group(1), [])
        elif line.startswith(".Lfunc_end"):
            cur = None
        elif cur is not None:
            s = line.split(";")[0].strip()
            if s and (not s.startswith(".") or s.endswith(":")):
                cur.append(s)
    return out


def early(instructions):
    """Instructions that come too early after a product, as (text, register)."""
    blocks, labels, block = [], {}, []
    for s in instructions:
        if s.endswith(":"):
            if block:
                blocks.append(block)
            block = []
            labels[s[:-1]] = len(blocks)
            continue
        block.append(s)
        if s.startswith(("s_cbranch", "s_branch", "s_endpgm")):
            blocks.append(block)
            block = []
    if block:
        blocks.append(block)

    def follow(n, state, found):
        state = dict(state)  # register -> [wait states since, needed]
        for s in blocks[n]:
            name, _, rest = s.replace("\t", " ").partition(" ")
            ops = [o.strip() for o in re.split(r",(?![^\[]*\])", rest)] if rest else []
            product = name.startswith("v_mfma")
            waits = int(ops[0], 0) + 1 if name == "s_nop" else 1
            if not name.startswith("s_"):
                store = "store" in name or name.startswith("ds_write") or \
                    (name.startswith("buffer_load") and s.endswith("lds"))
                dst = registers(ops[0]) if ops and not store else []
                src = registers(ops[1]) + registers(ops[2]) if product else \
                    [r for o in (ops if store else ops[1:]) for r in registers(o)]
                for r in src + ([] if product else dst):
                    if r in state and found is not None:
                        found.append((s, r))
                for r in dst:
                    state.pop(r, None)
            for r in list(state):
                since, need = state[r]
                if since + waits >= need:
                    del state[r]
                else:
                    state[r] = (since + waits, need)
            if product:
                need = 18 if "x2_f32" in name else 12
                for r in registers(ops[0]):
                    state[r] = (0, need)
        return state

    states, work = {0: {}}, [0]
    after = {}
    for n, b in enumerate(blocks):
        words, after[n] = b[-1].split(), []
        if words[0].startswith(("s_cbranch", "s_branch")) and labels.get(words[1], len(blocks)) < len(blocks):
            after[n].append(labels[words[1]])
        if not words[0].startswith(("s_branch", "s_endpgm")) and n + 1 < len(blocks):
            after[n].append(n + 1)
    while work:
        n = work.pop()
        out = follow(n, states[n], None)
        for m in after[n]:
            if m not in states:
                states[m] = dict(out)
                work.append(m)
                continue
            grew = False
            for r, v in out.items():
                if r not in states[m] or states[m][r][0] > v[0]:
                    states[m][r], grew = v, True
            if grew:
                work.append(m)
    found = []
    for n, state in states.items():
        follow(n, state, found)
    return found


def test_the_check_sees_an_early_read():
    code = ["v_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], v[24:27], v[0:15]", "s_cbranch_scc1 .L1",
            "s_nop 15", "v_mov_b32 v40, v15", "s_endpgm", ".L1:", "v_mov_b32 v41, v15", "s_endpgm"]
    assert early(code) == [("v_mov_b32 v41, v15", 15)]
    # the branch is one wait state, s_nop n is n + 1
    assert early(code[:6] + ["s_nop 9"] + code[6:]) == [("v_mov_b32 v41, v15", 15)]
    assert early(code[:6] + ["s_nop 10"] + code[6:]) == []


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
def test_attention_kernels(tmp_path):
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
    assert kernels > 100

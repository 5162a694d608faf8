"""No vector memory instruction of the library reads an SGPR within five wait states of a VALU
instruction that wrote it (CPU, no GPU needed: the built code objects are disassembled).

The hardware does not wait there. The compiler keeps the distance for loads that it emits, not for
those in inline asm: a kernel whose base address was a spilled SGPR, restored by v_readlane right
before the asm load, read a wrong address. Kernels that spill their bases copy them inside the asm
(ffa_common.h); this test holds all others to the distance. A load into LDS must also stay one wait
state behind the scalar write of M0, which holds its LDS address.
"""

from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from fastest_flash_attention_amd.kernels import _lib

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
WAIT = 5
_SREG = re.compile(r"\bs(?:(\d+)\b|\[(\d+):(\d+)\])")
_VMEM = re.compile(r"^(global|buffer|scratch|flat)_")


def _sregs(operand: str) -> set:
    regs = set()
    for one, lo, hi in _SREG.findall(operand):
        regs |= {int(one)} if one else set(range(int(lo), int(hi) + 1))
    return regs


def _valu_writes(op: str, operands: list) -> set:
    """SGPRs that a VALU instruction writes: v_readlane / v_readfirstlane and compares write their
    first operand, carries and divisions' flags the second."""
    if not op.startswith("v_") or op.startswith("v_mfma") or op.startswith("v_accvgpr"):
        return set()
    regs = _sregs(operands[0]) if operands else set()
    if len(operands) > 1 and re.match(r"v_(add|sub|subrev|addc|subb|mad|div)_", op) and operands[1].startswith("s["):
        regs |= _sregs(operands[1])
    return regs


def hazards(lines):
    """(kernel, distance, writer, reader) of every violation in a disassembly."""
    found, kernel, recent = [], "", []  # recent: (wait states it takes, SGPRs written by VALU, text)
    for line in lines:
        head = re.match(r"^[0-9a-f]+ <(.+)>:", line)
        if head:
            kernel, recent = head.group(1), []
            continue
        text = line.split("//")[0].strip()
        if not text or text.endswith(":") or "file format" in text or text.startswith("Disassembly"):
            continue
        op, _, rest = text.partition(" ")
        operands = [x.strip() for x in rest.split(",")]
        if _VMEM.match(op):
            reads, distance = _sregs(rest), 0
            for states, written, writer in reversed(recent):
                if distance >= WAIT:
                    break
                if written & reads:
                    found.append((kernel, distance, writer, text))
                    break
                distance += states
        states = int(operands[0], 0) + 1 if op == "s_nop" else 1
        recent.append((states, _valu_writes(op, operands), text))
        recent = recent[-WAIT:]
    return found


def m0_hazards(lines):
    """Loads into LDS right behind a scalar write of M0."""
    found, before = [], ""
    for line in lines:
        text = line.split("//")[0].strip()
        if not text:
            continue
        if "load_lds" in text and re.match(r"s_\S+ m0,", before):
            found.append((before, text))
        before = text
    return found


def test_scanner_finds_a_planted_m0_hazard():
    load = "global_load_lds_dwordx4 v1, s[4:5]"
    assert m0_hazards(["s_mov_b32 m0, s3", "", load]) == [("s_mov_b32 m0, s3", load)]
    assert not m0_hazards(["s_mov_b32 m0, s3", "s_nop 0", load])


def test_scanner_finds_planted_hazards():
    def snippet(*between):
        return ["0000 <k>:", "v_readlane_b32 s1, v167, 57", *between, "global_load_lds_dwordx4 v120, s[0:1]"]

    assert len(hazards(snippet())) == 1
    assert hazards(snippet("s_nop 3", ))[0][1] == 4 and not hazards(snippet("s_nop 4"))
    assert not hazards(snippet(*["v_mov_b32_e32 v1, v2"] * 5)) and hazards(snippet(*["v_mov_b32_e32 v1, v2"] * 4))
    assert not hazards(["0000 <k>:", "v_readlane_b32 s1, v167, 57", "s_mov_b64 s[8:9], s[0:1]",
                        "global_load_lds_dwordx4 v120, s[8:9]"])
    assert not hazards(["0000 <k>:", "s_add_u32 s0, s0, s2", "global_load_lds_dwordx4 v120, s[0:1]"])
    assert hazards(["0000 <k>:", "v_cmp_gt_i32_e64 s[4:5], s2, v3", "global_load_dword v1, v2, s[4:5]"])
    assert not hazards(snippet()[:2] + ["0010 <other>:"] + snippet()[2:])


def test_no_kernel_reads_a_fresh_sgpr(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("llvm-objdump not installed")
    _lib.load()
    lib = shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, capture_output=True, cwd=tmp_path)
    images = sorted(f for f in os.listdir(tmp_path) if f.endswith("gfx950"))
    assert len(images) >= 5
    loads, found = 0, []
    for f in images:
        out = subprocess.run([OBJDUMP, "-d", f], check=True, capture_output=True, text=True, cwd=tmp_path).stdout
        loads += out.count("global_load_lds_dwordx4")
        found += hazards(out.splitlines()) + m0_hazards(out.splitlines())
    assert loads > 1000
    assert not found, "\n".join(str(x) for x in found[:20])

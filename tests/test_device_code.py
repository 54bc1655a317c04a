"""The gfx950 code of the built library: a matrix product may read what a
vector instruction wrote two wait states ago at the earliest.  The compiler
keeps that distance for instructions of its own, not for those it was given as
assembly (v_fma_mixlo_f16 and v_fma_mixhi_f16 of the hi + lo split)."""
import os
import re
import shutil
import subprocess

import pytest

from nanoinfer_amd import build

OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
CSRC = os.path.join(os.path.dirname(os.path.abspath(build.__file__)), "csrc")
WAIT_STATES = 2


def _registers(operand):
    m = re.match(r"v\[(\d+):(\d+)\]$", operand)
    if m:
        return range(int(m[1]), int(m[2]) + 1)
    m = re.match(r"v(\d+)$", operand)
    return range(int(m[1]), int(m[1]) + 1) if m else ()


def close_pairs(lines):
    """(writes of the split, products that read one too early) of disassembled instructions."""
    written, at, writes, early = {}, 0, 0, []
    for line in lines:
        line = line.split("//")[0].strip()
        if not line or line.endswith(":") or line.startswith((".", ";")):
            continue
        op, _, rest = line.partition(" ")
        args = [x.strip() for x in rest.split(",")]
        if op == "s_nop":
            at += int(args[0], 0) + 1
            continue
        at += 1
        if op.startswith("v_fma_mix"):
            writes += 1
            for r in _registers(args[0]):
                written[r] = at
        elif op.startswith("v_mfma"):
            early += [line for x in args[1:3] for r in _registers(x)
                      if r in written and at - written[r] - 1 < WAIT_STATES]
            for r in _registers(args[0]):
                written.pop(r, None)
        elif op.startswith("v_"):  # the compiler's own write: it keeps the distance
            for r in _registers(args[0]):
                written.pop(r, None)
    return writes, early


def test_the_scan_finds_a_close_pair():
    mixhi = "\tv_fma_mixhi_f16 v74, v1, 1.0, -v3 op_sel:[0,0,1] op_sel_hi:[0,0,1]   // 000000001234: 01"
    mfma = "\tv_mfma_f32_16x16x16_f16 v[0:3], v[10:11], v[74:75], v[0:3]"
    other = "\tv_mul_f32_e32 v5, v6, v7"
    for between, found in (([], True), ([other], True), (["\ts_nop 0"], True), (["\ts_nop 1"], False),
                           ([other, other], False), (["\tv_mov_b32_e32 v74, v5"], False)):
        assert close_pairs([mixhi, *between, mfma]) == (1, [mfma.strip()] if found else [])
    assert close_pairs([mixhi, mfma.replace("v[74:75]", "v[76:77]")]) == (1, [])


def test_products_read_split_operands_in_time(tmp_path):
    if not os.path.exists(OBJDUMP) or not os.path.exists(build.LIB):
        pytest.skip("needs llvm-objdump and the built library")
    lib = shutil.copy(build.LIB, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, capture_output=True)
    total = 0
    for part in sorted(tmp_path.glob("*gfx950*")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(part)], check=True, capture_output=True,
                              text=True).stdout
        writes, early = close_pairs(text.splitlines())
        assert not early, f"{part.name}: {early[:3]}"
        total += writes
    assert total > 1000


def test_every_split_settles():
    """The distance above does not rest on the schedule: the split's results
    reach products through split4, split8 or settle()."""
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith((".hip", ".h")):
            continue
        text = open(os.path.join(CSRC, name)).read()
        for m in re.finditer(r"\bsplit_w16x2\((?!float)", text):
            after = text[m.start():m.start() + 1600]
            assert "settle(" in after, f"{name}:{text.count(chr(10), 0, m.start()) + 1}"

"""Global -> LDS copies of the built kernels (buffer_load ... lds) stand behind the wait states that gfx950 needs and that the
compiler adds only for copies it writes itself: one between a write of m0 and the copy that takes its LDS address from
there, five between a vector instruction's write of a scalar register and the copy that reads it (the buffer's base and
size). Without them a copy can use the place or the buffer of the copy before. Read from the disassembly of the library's
own kernels, along the code as it is laid out."""

import os
import re
import shutil
import subprocess

import pytest

from tensorpack_amd import _native

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
M0_STATES, SGPR_STATES = 1, 5


def _scalars(operand):
    m = re.match(r"s\[(\d+):(\d+)\]$", operand)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.match(r"s(\d+)$", operand)
    return {int(m[1])} if m else set()


def _short_waits(lines):
    """(copies, the copies that come too early) of a disassembly."""
    copies, early, past = 0, [], []                              # past: the last instructions, (name, operands)
    for line in lines:
        line = line.split("//")[0].split(";")[0].strip()
        if not line or line.endswith(":"):
            continue
        name, _, rest = line.partition(" ")
        operands = [x.strip() for x in rest.split(",")]
        if name.startswith("buffer_load") and "lds" in rest.split():
            copies += 1
            reads = set().union(*(_scalars(x.split()[0]) for x in operands if x))
            states = 0
            for before, its in reversed(past):
                if states >= SGPR_STATES:
                    break
                if its[0] == "m0" and states < M0_STATES or before.startswith("v_") and _scalars(its[0]) & reads:
                    early.append((line, states, before, its))
                states += int(its[0], 0) + 1 if before == "s_nop" else 1
        past = past[-8:] + [(name, operands)]
    return copies, early


def test_the_scan_sees_a_missing_wait():
    ok = ["s_mov_b32 m0, s3", "s_nop 0", "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"]
    assert _short_waits(ok) == (1, [])
    assert len(_short_waits([ok[0], ok[2]])[1]) == 1
    assert len(_short_waits(["v_readfirstlane_b32 s5, v2", "s_nop 1"] + ok)[1]) == 1
    assert _short_waits(["v_readfirstlane_b32 s5, v2", "s_nop 2"] + ok) == (1, [])
    assert _short_waits(["v_readfirstlane_b32 s8, v2"] + ok) == (1, [])


def test_copies_into_lds_wait(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no disassembler here")
    lib = shutil.copy(_native.HIP_LIB_PATH, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, capture_output=True, cwd=tmp_path)
    copies = 0
    for name in sorted(os.listdir(tmp_path)):
        if "gfx950" not in name:
            continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(tmp_path / name)], check=True,
                              capture_output=True, text=True).stdout
        n, early = _short_waits(text.splitlines())
        assert not early, (name, len(early), early[:3])
        copies += n
    assert copies > 0

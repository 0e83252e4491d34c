"""Copies of single words into LDS (global_load_lds) of the built kernels stand behind a wait state after m0, which holds their place there, is
written (see test_copy_waits, whose copies take scalar registers too). Read from the disassembly of the library's own kernels."""

import os
import shutil
import subprocess

import pytest

from tensorpack_amd import _native
from test_copy_waits import OBJDUMP


def _short_waits(lines):
    """(copies, the copies that come too early): states since m0 was written, along the code as it is laid out."""
    copies, early, states = 0, [], None
    for line in lines:
        line = line.split("//")[0].split(";")[0].strip()
        name, _, rest = line.partition(" ")
        if not rest and name != "s_nop":
            continue
        if name.startswith("global_load_lds"):
            copies += 1
            if states is not None and states < 1:
                early.append(line)
        if rest.split(",")[0].strip() == "m0":
            states = 0
        elif states is not None:
            states += int(rest, 0) + 1 if name == "s_nop" else 1
    return copies, early


def test_the_scan_sees_a_missing_wait():
    assert _short_waits(["s_mov_b32 m0, s3", "s_nop 0", "global_load_lds_dword v[0:1], off"]) == (1, [])
    assert len(_short_waits(["s_mov_b32 m0, s3", "global_load_lds_dword v[0:1], off"])[1]) == 1


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

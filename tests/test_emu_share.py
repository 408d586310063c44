"""The split of attention batches over workers (cx_share.hpp) compiled for the
host, with the address and undefined-behaviour checks, and walked as the kernel
walks it on random batches: decode, thousands of sequences, verify rounds,
prompts, mixtures, lengths at the type's ends (tests/emu/share_check.cpp)."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "chenxing_amd", "csrc")

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    tmp = tmp_path_factory.mktemp("share")
    os.makedirs(tmp / "hip")
    shutil.copy(os.path.join(HERE, "emu", "hip_emu.h"), tmp / "hip" / "hip_runtime.h")
    out = str(tmp / "share_check")
    r = subprocess.run(["g++", "-std=c++20", "-O1", "-g", "-fsanitize=address,undefined",
                        "-fno-sanitize-recover=undefined", "-pthread", "-I", str(tmp), "-I", CSRC,
                        "-include", "hip/hip_runtime.h", os.path.join(HERE, "emu", "share_check.cpp"),
                        "-o", out], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    return out


@pytest.mark.parametrize("seed", range(3))
def test_every_unit_is_in_one_piece(exe, seed):
    r = subprocess.run([exe, "250", str(seed)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout + r.stderr[-3000:]

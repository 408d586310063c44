"""The kernels' dynamic-LDS limits (cx_lds.hpp) on the host, against a HIP of the
test's own (tests/emu/lds_check.cpp)."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "chenxing_amd", "csrc")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_limits_by_device(tmp_path):
    os.makedirs(tmp_path / "hip")
    (tmp_path / "hip" / "hip_runtime.h").write_text("")
    exe = str(tmp_path / "lds_check")
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=thread", "-pthread", "-I",
                        str(tmp_path), "-I", CSRC, os.path.join(HERE, "emu", "lds_check.cpp"), "-o",
                        exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout + r.stderr[-3000:]

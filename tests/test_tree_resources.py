"""The tree operators' and the 4-bit products' kernels, compiled for gfx950, run
without a scratch frame and without out-of-line calls, two waves of 256 registers a
SIMD (CPU only: device-only compilation to assembly)."""
from __future__ import annotations

import os
import re
import tempfile

import pytest

from test_kernel_resources import HIPCC, _asm

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")


@pytest.mark.parametrize("src,least", [("cx_walk.hip", 2), ("cx_tree.hip", 42), ("cx_w4.hip", 66)])
def test_kernels_have_no_scratch_and_no_calls(src, least):
    with tempfile.TemporaryDirectory() as tmp:
        s = _asm(src, os.path.join(tmp, "k.s"))
    kernels = re.findall(r"\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", s, re.S)
    assert len(kernels) >= least

    def field(body, name):
        return int(re.search(rf"\.amdhsa_{name}\s+(\d+)", body).group(1))
    funcs = set(re.findall(r"\.type\s+(\S+),@function", s))
    assert not {r for r in re.findall(r"(\S+)@rel32@lo", s) if r in funcs}
    for name, body in kernels:
        assert field(body, "private_segment_fixed_size") == 0, name
        assert field(body, "next_free_vgpr") <= 256, name

"""The paged cache's kernels, compiled for gfx950, run without a scratch frame
and without out-of-line calls (CPU only: device-only compilation to assembly),
and the attention tiles fit the waves per SIMD that their launches count on."""
from __future__ import annotations

import os
import re
import tempfile

import pytest

from test_kernel_resources import HIPCC, _asm

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="needs hipcc")


@pytest.mark.parametrize("src", ["cx_kv.hip", "cx_attend.hip"])
def test_kernels_have_no_scratch_and_no_calls(src):
    with tempfile.TemporaryDirectory() as tmp:
        s = _asm(src, os.path.join(tmp, "k.s"))
    kernels = re.findall(r"\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", s, re.S)
    assert len(kernels) >= 13

    def field(body, name):
        return int(re.search(rf"\.amdhsa_{name}\s+(\d+)", body).group(1))
    funcs = set(re.findall(r"\.type\s+(\S+),@function", s))
    assert not {r for r in re.findall(r"(\S+)@rel32@lo", s) if r in funcs}
    for name, body in kernels:
        assert field(body, "private_segment_fixed_size") == 0, name
        m = re.search(r"attend_splitILi(\d+)ELi(\d+)ELb(\d)", name)
        if m:
            D, NT, F8 = map(int, m.groups())
            waves = (3 if F8 else 4) if D * NT == 64 else \
                2 if D * NT < 256 or (NT == 2 and not F8) else 1
            regs = field(body, "next_free_vgpr")     # AGPRs included, of 512 a SIMD lane
            assert -(-regs // 8) * 8 * waves <= 512, (name, regs, waves)

"""Products with 4-bit weights that run a split's steps to the end of a long K, against
their restatement (oracle/w4_ref.py), whose bound one lost tile passes."""
from __future__ import annotations

import pytest

import paged_cases as C
from test_gpu_w4 import _check, _inputs

pytestmark = pytest.mark.gpu

# (rows, N, K, group): eight waves a row of W and 32 rows of W a wave (N of 4097 to 8192, 17 to
# 32 rows), the splits beside it, and K that ends in a tile
DEEP = [(20, 4112, 4096, 32), (32, 4112, 4128, 32), (20, 6144, 4096, 128), (32, 6144, 4160, 64),
        (17, 8192, 4096, 64), (32, 8192, 4128, 32), (29, 5000, 8320, 128), (24, 4096, 4096, 64),
        (32, 8200, 4096, 32), (64, 4112, 4160, 64), (61, 2048, 8192, 128), (33, 512, 14336, 32),
        (9, 6144, 4128, 32)]


@pytest.mark.parametrize("shift", [False, True])
@pytest.mark.parametrize("M,N,K,group", DEEP)
def test_linear(M, N, K, group, shift):
    import torch
    from chenxing_amd import w4
    from chenxing_amd._lib import w4_linear_device
    x, codes, scale, sh = _inputs(M, N, K, group, shift)
    tiles, scales = w4.pack(*(None if t is None else torch.from_numpy(t).cuda()
                              for t in (codes, scale, sh)))
    for dtype in (torch.float32, torch.bfloat16):
        got = w4_linear_device(C.to_gpu(x), tiles, scales, N, dtype)
        _check(x, codes, scale, sh, got, dtype == torch.bfloat16)

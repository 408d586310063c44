"""The attention entry point on the host: its workspace (one of the largest call
serves every smaller one) and its scores' range (CPU)."""
from __future__ import annotations

import os

import pytest

from chenxing_amd import _lib
from test_paged_api import A, _attend, _kv

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH),
                                reason="libcx_sampler.so not built")


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("heads", [(32, 8), (28, 4), (8, 8), (40, 1)])
def test_bytes_grow_with_the_new_tokens(D, heads):
    size = _lib.load().cx_paged_attention_workspace_bytes
    last = 0
    for new in [*range(1, 200), 1000, 4096, 2 ** 28, 2 ** 31 - 1]:
        n = size(*heads, D, new)
        assert n >= last, (new, n, last)
        last = n
    for q in range(heads[1], heads[0], heads[1]):
        assert size(q, heads[1], D, 7) <= size(*heads, D, 7)


@pytest.mark.parametrize("dtype,stride", [(1, 2 * 4096 * 2), (3, 2 * (4096 + 128))])
def test_a_workspace_of_the_most_new_tokens_serves_fewer(dtype, stride):
    """Calls without rows in their table's pages get as far as the size's check, and
    no further: n_pages past the table is refused after it."""
    lib = _lib.load()
    for most in (5, 9, 17):
        need = lib.cx_paged_attention_workspace_bytes(4, 2, 128, most)
        for new in range(1, most + 1):
            kv = _kv(dtype=dtype, stride=stride, M=1 << 22, ld=1 << 22, T=1 << 22)
            assert _attend(kv, new=new, nbytes=need) == _lib.CX_EINVAL
            assert b"too many tokens" in lib.cx_last_error()


@pytest.mark.parametrize("bad", [dict(scale=float("inf")), dict(scale=1e39), dict(cap=1e-45),
                                 dict(scale=1e20, cap=1e-20)], ids=str)
def test_scores_past_the_range_of_fp32_are_refused(bad):
    assert _attend(_kv(), **bad) == _lib.CX_EINVAL and b"fp32" in _lib.load().cx_last_error()


@pytest.mark.parametrize("off", [1, 4, 8])
def test_a_workspace_off_16_bytes_is_refused(off):
    assert _attend(_kv(), ws=A + off) == _lib.CX_EINVAL
    assert b"workspace" in _lib.load().cx_last_error()

"""The 4-bit products' oracle: its sums by closed forms, and a bound on a device
result's error that a lost piece of K passes (CPU only)."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import w4_ref as R
from oracle.bf16 import bf16_bits_to_f32
from test_gpu_w4 import SIZES, _inputs
from test_gpu_w4_depths import DEEP


def _case(M, N, K, group, shift):
    N = min(N, 256)                                # (each row of W has its own bound)
    x, codes, scale, sh = _inputs(M, N, K, group, shift)
    return bf16_bits_to_f32(x).astype(np.float64), codes, scale, sh


@pytest.mark.parametrize("shift", [False, True])
@pytest.mark.parametrize("M,N,K,group", sorted({*SIZES, *DEEP}))
def test_a_lost_piece_passes_the_bound(M, N, K, group, shift):
    """32 k of one group, or a tile of 128, left out or taken twice: more than half of all
    results are further off than the bound, in fp32 and in bf16."""
    x, codes, scale, sh = _case(M, N, K, group, shift)
    w = R.weights(codes, scale, sh)
    for bf16 in (False, True):
        y, tol = R.linear(x, codes, scale, sh, bf16)
        assert np.abs(y - x @ w.T).max() <= 1e-9 * np.abs(y).max() + 1e-12
        for size in (32, 128):
            for k in sorted({0, (K - 1) // size // 2 * size, (K - 1) // size * size}):
                piece = x[:, k:k + size] @ w[:, k:k + size].T
                assert (np.abs(piece) > tol).mean() > 0.5, (bf16, size, k)


def test_the_bound_holds_for_sums_in_any_order():
    """fp32 sums of the terms, one after the other, backwards and by halves."""
    rng = np.random.default_rng(1)
    for K, group, shift, offset in ((256, 64, True, 0.0), (256, 32, False, 0.0), (512, 128, True, 30.0)):
        x, codes, scale, sh = _inputs(4, 24, K, group, shift, 2, offset)
        x = bf16_bits_to_f32(x)
        y, tol = R.linear(x.astype(np.float64), codes, scale, sh)
        c = np.float32(1.0 if shift else 1.5)
        v = (1 + codes / 16.0).astype(np.float32)
        for order in range(4):
            out = np.zeros(y.shape, np.float32)
            for g in range(K // group):
                ks = np.arange(g * group, (g + 1) * group)
                ks = ks if order == 0 else ks[::-1] if order == 1 else rng.permutation(ks)
                P, H = np.zeros(y.shape, np.float32), np.zeros(y.shape, np.float32)
                for k in ks:
                    P = P - c * x[:, k:k + 1]
                    H = H + x[:, k:k + 1] / np.float32(16)
                for k in ks[::-1] if order == 3 else ks:
                    P = P + x[:, k:k + 1] * v[:, k]
                if shift:
                    out = out + sh[:, g].astype(np.float32) * H
                out = out + scale[:, g].astype(np.float32) * P
            assert (np.abs(16.0 * out - y) <= tol).all()

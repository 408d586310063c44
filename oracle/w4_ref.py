"""CPU restatement in 64 bits of the products with 4-bit weights: the oracle of
cx_w4_linear_bf16.  Test infrastructure only.

W[n, k] = scale * code + shift, or scale * (code - 8); the tiles' format is that of
include/cx_sampler.h.
"""
from __future__ import annotations

import numpy as np

from .paged_ref import U16, U32


def pack(codes, scale, shift=None):
    """(tiles int32, scales fp16) of codes [N, K], scale and shift [N, K / group]."""
    N, K = codes.shape
    n16, k128 = -(-N // 16), -(-K // 128)
    full = np.zeros((16 * n16, 128 * k128), np.uint32)
    full[:N, :K] = codes
    tiles = np.zeros((n16, k128, 64, 4), np.uint32)
    for j in range(4):
        for s in range(4):
            for e in range(8):
                k = 32 * s + 8 * j + e
                part = full[:, k::128].reshape(n16, 16, k128).transpose(0, 2, 1)
                tiles[:, :, 16 * j:16 * j + 16, s] |= part << np.uint32(4 * (e // 2) + 16 * (e % 2))
    both = scale[..., None] if shift is None else np.stack([scale, shift], 2)
    laid = np.zeros((16 * n16, *both.shape[1:]), np.float16)
    laid[:N] = both
    laid = laid.reshape(n16, 16, *both.shape[1:]).swapaxes(1, 2)
    return tiles.view(np.int32), np.ascontiguousarray(laid[..., 0] if shift is None else laid)


def weights(codes, scale, shift=None):
    N, K = codes.shape
    q = codes.reshape(N, scale.shape[1], -1).astype(np.float64)
    s = scale.astype(np.float64)[..., None]
    w = s * (q - 8) if shift is None else s * q + shift.astype(np.float64)[..., None]
    return w.reshape(N, K)


def linear(x, codes, scale, shift=None, bf16=False):
    """(y [M, N], bound on a device result's error): fp32 sums, in any order, of the
    terms 16 s (1 + q / 16) x and (t - 16 s) x."""
    N, K = codes.shape
    y = x @ weights(codes, scale, shift).T
    s = np.repeat(np.abs(scale.astype(np.float64)), K // scale.shape[1], 1)
    t = 8 * s if shift is None else np.repeat(np.abs(shift.astype(np.float64)), K // scale.shape[1], 1)
    mag = np.abs(x) @ (s * (codes + 16.0) + t + 16 * s).T
    # K products (exact) and their sums, a group's two scalings and sums
    tol = (K + 2 * scale.shape[1] + 8) * U32 * mag + 1e-38
    if bf16:
        tol = tol + U16 * 1.01 * (np.abs(y) + tol)
    return y, tol

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
    """(y [M, N], bound on a device result's error).

    y / 16 = sum over groups g of s_g P_g + t_g H_g, with P_g = sum x (1 + q / 16) - c
    sum x and H_g = sum x / 16 of the group's k; c = 1, without shifts 1.5 and t = 0.
    The products of bf16 are exact in fp32.  In whatever order a group's are summed,
    each of them passes through one addition at least, so that at most 2 group
    additions' roundings, of partial sums below A_g = sum |x| (1 + q / 16 + c), are in
    P_g, and group, below sum |x| / 16, in H_g.  Each group enters the sum of groups with
    two roundings, and that may be split into 8 which add up with 7 more: of partial
    sums below the sum of the groups' |s P| + |t H|, which do not grow as the sums of
    magnitudes do.  (1.01: the roundings' own products.)"""
    N, K = codes.shape
    M, groups = x.shape[0], scale.shape[1]
    g = K // groups
    y = x @ weights(codes, scale, shift).T
    s = np.abs(scale.astype(np.float64)).T
    t = np.zeros_like(s) if shift is None else np.abs(shift.astype(np.float64)).T
    c = 1.5 if shift is None else 1.0
    inside, between = np.zeros((M, N)), np.zeros((M, N))
    for i in range(groups):                    # (a group at a time: M N K values are many)
        xg = x[:, i * g:(i + 1) * g]
        v = 1 + codes[:, i * g:(i + 1) * g].T / 16.0
        mag = np.abs(xg)
        inside += 2 * g * s[i] * (mag @ (v + c)) + g * t[i] * mag.sum(1, keepdims=True) / 16
        between += s[i] * np.abs(xg @ (v - c)) + t[i] * np.abs(xg.sum(1, keepdims=True)) / 16
    between += U32 * 1.01 * inside
    tol = 16 * U32 * 1.01 * (inside + (2 * groups + 7) * between) + 1e-38
    if bf16:
        tol = tol + U16 * 1.01 * (np.abs(y) + tol)
    return y, tol

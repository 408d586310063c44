"""CPU restatement of the paged KV-cache operators in 64 bits: the oracle of
cx_kv_append_bf16, cx_paged_attention_bf16 and cx_kv_copy_pages.  Test
infrastructure only.

Reference: RMSNorm, RoPE and YaRN (chenxing/core/tensor.py:36-180), causal
grouped-query attention with a sliding window (chenxing/core/attention.py
:43-148), the paged cache (chenxing/engine/radix_kv.py:74-273).  The softmax
cap, the per-head norms and the 8-bit cache are this library's; the formulas
are those of include/cx_sampler.h.

A layer's pages are numpy arrays of raw bits here: uint16 [n, heads, 2 P D]
(bf16) or uint8 [n, heads, 2 P D + 8 P] (e4m3).
"""
from __future__ import annotations

import numpy as np

from .bf16 import bf16_bits_to_f32

U32 = 2.0 ** -24                      # unit roundoff of fp32
U16 = 2.0 ** -8                       # of bf16 (8 significant bits)


def e4m3_values() -> np.ndarray:
    """The 256 codes' values: sign, 4 exponent bits (bias 7), 3 of mantissa;
    0x7F and 0xFF are NaN, there is no infinity."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    x = np.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * 2.0 ** (e - 7.0))
    x = np.where((c & 0x7F) == 0x7F, np.nan, x)
    return np.where(c & 0x80, -x, x)


E4M3 = e4m3_values()


def e4m3_codes(x: np.ndarray) -> np.ndarray:
    """The codes of the nearest values, ties to the even code, saturating."""
    v = E4M3[:0x7F]
    a = np.abs(np.asarray(x, np.float64))
    i = np.clip(np.searchsorted(v, a), 1, 0x7E)
    lo, hi = v[i - 1], v[i]
    up = (a - lo > hi - a) | ((a - lo == hi - a) & (i % 2 == 0))
    code = np.where(a >= v[-1], 0x7E, np.where(up, i, i - 1)).astype(np.uint8)
    return np.where(np.signbit(x), code | 0x80, code).astype(np.uint8)


def _at(P: int, D: int, E: int, o, d):
    """Element offsets of K and V of the page's token o at dim d."""
    return ((d // E) * P + o) * E + d % E, P * D + ((o // E) * D + d) * E + o % E


def pack(k: np.ndarray, v: np.ndarray, ks=None, vs=None) -> np.ndarray:
    """Pages of dense [n, heads, P, D] bits (uint16 bf16; uint8 e4m3 with the
    scales [n, heads, P])."""
    n, H, P, D = k.shape
    E = 8 if k.dtype == np.uint16 else 16
    o, d = np.meshgrid(np.arange(P), np.arange(D), indexing="ij")
    ka, va = _at(P, D, E, o, d)
    out = np.zeros((n, H, 2 * P * D), k.dtype)
    out[:, :, ka] = k
    out[:, :, va] = v
    if ks is None:
        return out
    sc = np.concatenate([ks, vs], 2).astype(np.float32)
    return np.concatenate([out, sc.view(np.uint8)], 2)


def unpack(pages: np.ndarray, D: int):
    """(K, V) as fp64 [n, heads, P, D]: the values the pages stand for."""
    n, H, width = pages.shape
    bf16 = pages.dtype == np.uint16
    E = 8 if bf16 else 16
    P = width // (2 * D if bf16 else 2 * D + 8)
    o, d = np.meshgrid(np.arange(P), np.arange(D), indexing="ij")
    ka, va = _at(P, D, E, o, d)
    if bf16:
        x = bf16_bits_to_f32(pages).astype(np.float64)
        return x[:, :, ka], x[:, :, va]
    x = E4M3[pages[:, :, :2 * P * D]]
    sc = np.ascontiguousarray(pages[:, :, 2 * P * D:]).view(np.float32).astype(np.float64)
    with np.errstate(invalid="ignore"):
        return x[:, :, ka] * sc[:, :, :P, None], x[:, :, va] * sc[:, :, P:, None]


def places(kv_len, q_start, P: int, M: int, table, n_pages: int):
    """(sequence, position, page or -1, place in the page) of every new token."""
    out = []
    for b in range(len(kv_len)):
        n = q_start[b + 1] - q_start[b]
        for i in range(n):
            p = int(kv_len[b]) - n + i
            pg = int(table[b][p // P]) if 0 <= p < M * P else -1
            out.append((b, p, pg if 0 <= pg < n_pages else -1, p % P))
    return out


def norm(x, w, eps):
    if w is None:
        return x
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def rotate(x, pos, rope, interleaved):
    """x [T, heads, D] at positions pos [T]; rope [positions, r] (cosines, sines)."""
    if rope is None:
        return x
    r = rope.shape[1]
    cs = rope[np.clip(pos, 0, len(rope) - 1)].astype(np.float64)
    c, s = cs[:, None, :r // 2], cs[:, None, r // 2:]
    y = x.copy()
    ia, ib = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2),
                                                                  slice(r // 2, r))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def attend(q, K, V, table, kv_len, q_start, P, scale, window=0, softcap=0.0):
    """(out [T, Hq, D], bound on a device result's error) in fp64.

    q [T, Hq, D]; K, V [n, heads, P, D].  The bound: fp32 products and sums
    (the scores' over D, the output's over the tokens, each in any order), a
    few roundings of the scores and of exp2, softmax terms taken as two bf16
    parts, one rounding of the result to bf16.
    """
    T, Hq, D = q.shape
    n_pages, H = K.shape[:2]
    G, M = Hq // H, np.shape(table)[1]
    out, tol = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    pl = places(kv_len, q_start, P, M, table, n_pages)
    for t, (b, pos, _, _) in enumerate(pl):
        s = np.arange(max(0, pos - window + 1) if window else 0, min(pos + 1, M * P))
        pg = np.asarray(table[b])[s // P].astype(np.int64) if len(s) else s
        keep = (pg >= 0) & (pg < n_pages)
        pg, o = pg[keep], s[keep] % P
        if not len(pg):
            continue
        for h in range(Hq):
            k, v = K[pg, h // G, o], V[pg, h // G, o]
            with np.errstate(all="ignore"):
                x = k @ q[t, h] * scale
                mag = np.abs(k) @ np.abs(q[t, h]) * scale
                if softcap:
                    x = softcap * np.tanh(x / softcap)
                e = np.exp(x - x.max())
                p = e / e.sum()
                o_ = p @ v
                ds = 2 * (D + 64) * U32 * mag + 8 * U32 * (np.abs(x) + np.abs(x.max()) + softcap)
                rel = 2 * ds + (2 * len(x) + 64) * U32 + 2.0 ** -16
                a = p @ (np.abs(v) * rel[:, None]) + np.abs(o_) * (p @ rel)
            out[t, h] = o_
            tol[t, h] = a + (U16 * 1.01) * (np.abs(o_) + a) + 1e-38
    return out, tol

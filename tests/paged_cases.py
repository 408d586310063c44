"""Inputs of the paged KV-cache tests: pages, tables and batches as numpy
arrays, with NaN in every place that no sequence holds."""
from __future__ import annotations

import numpy as np

from oracle import paged_ref as R
from oracle.bf16 import f32_to_bf16_bits

NAN16, NAN8 = 0x7FC0, 0x7F


def dense_pages(rng, n, H, P, D, cache, std=1.0):
    """(K, V, k scales, v scales): dense bits of random pages."""
    k, v = (rng.normal(0, std, (n, H, P, D)).astype(np.float32) for _ in range(2))
    if cache == "bf16":
        return f32_to_bf16_bits(k), f32_to_bf16_bits(v), None, None
    ks, vs = (np.abs(x).max(3).astype(np.float32) / np.float32(448) for x in (k, v))
    return (R.e4m3_codes(k / ks[..., None]), R.e4m3_codes(v / vs[..., None]), ks, vs)


def batch(rng, lens, new, P, spare=3, width=None):
    """A table whose pages are in random order, and the other pages' ids.
    Entries past a sequence's pages hold ids outside the pool."""
    need = [-(-max(0, n) // P) for n in lens]
    M = max(need + [1]) if width is None else width
    n = sum(need) + spare
    order = rng.permutation(n).astype(np.int32)
    table = rng.choice(np.array([-1, -7, n, n + 5, 2 ** 31 - 1]), (len(lens), M)).astype(np.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return table, np.asarray(lens, np.int32), q_start, n


def poison(K, V, ks, vs, table, lens, P):
    """NaN in every token that no sequence holds."""
    n = K.shape[0]
    free = np.ones((n, P), bool)
    for b, m in enumerate(lens):
        for s in range(m):
            free[table[b, s // P], s % P] = False
    bad = NAN16 if K.dtype == np.uint16 else NAN8
    for x in (K, V):
        x.transpose(0, 2, 1, 3)[free] = bad
    for x in (ks, vs):
        if x is not None:
            x.transpose(0, 2, 1)[free] = np.nan


def to_gpu(bits):
    """bf16 bits (uint16) as torch.bfloat16, anything else as it is."""
    import torch
    a = np.ascontiguousarray(bits)
    if a.dtype == np.uint16:
        return torch.from_numpy(a.view(np.int16)).cuda().view(torch.bfloat16)
    return torch.from_numpy(a).cuda()


def bits_of(t):
    import torch
    if t.dtype == torch.bfloat16:
        return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)
    return t.contiguous().cpu().numpy()

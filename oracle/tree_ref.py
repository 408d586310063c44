"""CPU restatement of the tree operators in 64 bits and whole numbers: the oracle of
cx_tree_attention_bf16, cx_tree_masks, cx_tree_accept and cx_kv_commit.  Test
infrastructure only.

The reference drafts chains (chenxing/engine/speculative.py); trees of drafts and
what they need of a cache are this library's, by the formulas of
include/cx_sampler.h.
"""
from __future__ import annotations

import numpy as np

from .paged_ref import U16, U32


def masks(parents, words: int, window: int = 0):
    """(mask [n, words] uint64, depth [n]) of one tree: the bits of a node and of its
    ancestors, with a window of those whose depth is above the node's less the window."""
    n = len(parents)
    m, d = np.zeros((n, words), np.uint64), np.zeros(n, np.int64)
    way = []
    for i, p in enumerate(parents):
        up = way[p] if 0 <= p < i else []
        way.append([*up, i])
        d[i] = len(up)
        for j in way[i]:
            if j < 64 * words and (not window or d[j] > d[i] - window):
                m[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return m, d


def accept(parents, tokens, sampled, width: int):
    """(path, next) of one tree."""
    if not len(parents):
        return [], -1
    path = [0]
    while len(path) < width:
        c = path[-1]
        kids = [i for i in range(c + 1, len(parents)) if parents[i] == c and tokens[i] == sampled[c]]
        if not kids:
            break
        path.append(kids[0])
    return path, int(sampled[path[-1]])


def moves(path, count, n: int, base: int):
    """[(from, to)] slots of one sequence's row of path."""
    out, last = [], -1
    for j, p in enumerate(list(path)[:max(count, 0)]):
        if p <= last or p >= n or base < 0:
            break
        last = p
        out.append((base + p, base + j))
    return out


def commit(K, V, ks, vs, table, kv_len, q_start, path, count, P: int):
    """Dense pages [.., n_pages, heads, P, D] (scales [.., n_pages, heads, P] or None)
    after the moves, in place."""
    n_pages, M = K.shape[-4], table.shape[1]

    def at(b, s):
        pg = int(table[b][s // P]) if s < M * P else -1
        return (pg, s % P) if 0 <= pg < n_pages else None
    for b in range(len(kv_len)):
        n = int(q_start[b + 1] - q_start[b])
        todo = [(at(b, s), at(b, d)) for s, d in
                moves(path[b], path.shape[1] if count is None else min(int(count[b]), path.shape[1]),
                      n, int(kv_len[b]) - n)]
        for x in (K, V, ks, vs):
            if x is None:
                continue
            old = x.copy()
            for s, d in todo:
                if s and d:
                    if x.ndim == K.ndim:
                        x[..., d[0], :, d[1], :] = old[..., s[0], :, s[1], :]
                    else:
                        x[..., d[0], :, d[1]] = old[..., s[0], :, s[1]]


def allowed(table, kv_len, q_start, mask, depth, P: int, n_pages: int, window: int):
    """(sequence, slots) that each new token attends to."""
    out = []
    M = np.shape(table)[1]
    for b in range(len(kv_len)):
        n = int(q_start[b + 1] - q_start[b])
        base = max(int(kv_len[b]), 0) - n
        for i in range(n):
            row = int(q_start[b]) + i
            s = np.arange(min(max(int(kv_len[b]), 0), M * P))
            node = s - base
            ok = node < 0
            if window:
                ok &= s > base + int(depth[row]) - window
            word = np.clip(node // 64, 0, mask.shape[1] - 1)
            bit = (mask[row][word] >> (node % 64).astype(np.uint64)) & np.uint64(1)
            ok |= (node >= 0) & (node < 64 * mask.shape[1]) & (bit > 0)
            s = s[ok]
            pg = np.asarray(table[b])[s // P].astype(np.int64)
            out.append((b, s[(pg >= 0) & (pg < n_pages)]))
    return out


def attend(q, K, V, table, kv_len, q_start, mask, depth, P, scale, window=0, softcap=0.0):
    """(out [T, Hq, D], bound on a device result's error) in fp64, as
    paged_ref.attend: fp32 products and sums, a few roundings of the scores and of
    exp2, softmax terms as two bf16 parts, one rounding of the result to bf16."""
    T, Hq, D = q.shape
    n_pages, H = K.shape[:2]
    G = Hq // H
    out, tol = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    for t, (b, s) in enumerate(allowed(table, kv_len, q_start, mask, depth, P, n_pages, window)):
        if not len(s):
            continue
        pg, o = np.asarray(table[b])[s // P].astype(np.int64), s % P
        for h in range(Hq):
            k, v = K[pg, h // G, o], V[pg, h // G, o]
            with np.errstate(all="ignore"):
                x = k @ q[t, h] * scale
                mag = np.abs(k) @ np.abs(q[t, h]) * scale
                if softcap and np.isfinite(softcap):
                    x = softcap * np.tanh(x / softcap)
                e = np.exp(x - x.max())
                p = e / e.sum()
                o_ = p @ v
                cap = min(softcap, 256.0)      # a larger cap's error goes with the score
                ds = 2 * (D + 64) * U32 * mag + 32 * U32 * (np.abs(x) + np.abs(x.max())) + 8 * U32 * cap
                rel = 2 * ds + (2 * len(x) + 64) * U32 + 2.0 ** -16
                a = p @ (np.abs(v) * rel[:, None]) + np.abs(o_) * (p @ rel)
            out[t, h] = o_
            tol[t, h] = a + (U16 * 1.01) * (np.abs(o_) + a) + 1e-38
    return out, tol

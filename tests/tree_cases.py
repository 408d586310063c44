"""Inputs of the tree operators' tests: trees, masks and batches as numpy arrays."""
from __future__ import annotations

import numpy as np

import paged_cases as C
from oracle import paged_ref as R
from oracle import tree_ref as Q
from oracle.bf16 import f32_to_bf16_bits

ATTEND = {
    # name: cache, Hq, Hkv, D, P, lengths, nodes, words, window, softcap, kind of masks
    "one_node": ("bf16", 4, 2, 64, 16, [1], [1], 1, 0, 0.0, "tree"),
    "one_node_later": ("bf16", 4, 2, 128, 16, [40], [1], 1, 0, 0.0, "tree"),
    "only_nodes": ("bf16", 8, 2, 128, 16, [7, 16, 33], [7, 16, 33], 1, 0, 0.0, "tree"),
    "edges": ("bf16", 8, 2, 128, 16, [15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129],
              [5, 5, 17, 1, 2, 3, 31, 32, 33, 9, 9, 9], 1, 0, 0.0, "tree"),
    "edges_e4m3": ("e4m3", 8, 2, 128, 16, [15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129],
                   [5, 5, 17, 1, 2, 3, 31, 32, 33, 9, 9, 9], 1, 0, 0.0, "tree"),
    "none_and_some": ("bf16", 4, 2, 128, 16, [0, 20, 5, 90], [0, 0, 5, 12], 1, 0, 0.0, "tree"),
    "full": ("bf16", 32, 8, 128, 16, [300, 64], [64, 64], 1, 0, 0.0, "tree"),
    "full_e4m3": ("e4m3", 32, 8, 128, 32, [300, 64], [64, 64], 1, 0, 0.0, "tree"),
    "words": ("bf16", 4, 1, 64, 16, [200, 391], [130, 129], 3, 0, 0.0, "tree"),
    "past_the_words": ("bf16", 4, 2, 64, 16, [100, 170], [80, 70], 1, 0, 0.0, "tree"),
    "any_bits": ("bf16", 6, 2, 128, 16, [80, 41, 30], [37, 20, 30], 1, 0, 0.0, "bits"),
    "empty_rows": ("bf16", 4, 2, 128, 16, [9, 30, 70], [9, 30, 64], 1, 0, 0.0, "sparse"),
    "empty_rows_e4m3": ("e4m3", 4, 2, 64, 16, [9, 30, 70], [9, 30, 64], 1, 0, 0.0, "sparse"),
    "chain": ("bf16", 8, 2, 128, 16, [300, 50], [9, 17], 1, 0, 0.0, "chain"),
    "window": ("bf16", 8, 2, 128, 16, [40, 100, 333, 700], [12, 25, 33, 64], 1, 50, 0.0, "tree"),
    "window_one": ("bf16", 4, 2, 64, 16, [40, 100], [12, 25], 1, 1, 0.0, "tree"),
    "window_e4m3": ("e4m3", 4, 2, 256, 32, [5, 700, 1300], [5, 20, 25], 1, 333, 50.0, "tree"),
    "deep_window": ("bf16", 4, 4, 64, 16, [60, 200], [50, 64], 1, 7, 0.0, "chain"),
    "softcap": ("bf16", 4, 2, 128, 16, [300, 60], [20, 33], 1, 0, 5.0, "tree"),
    "softcap_wide": ("bf16", 4, 2, 128, 16, [300, 60], [20, 33], 1, 0, 1000.0, "tree"),
    "wide_heads": ("bf16", 6, 3, 256, 32, [90, 300], [33, 64], 1, 0, 0.0, "tree"),
    "wide_heads_e4m3": ("e4m3", 8, 1, 256, 16, [90, 513], [33, 64], 1, 0, 0.0, "tree"),
    "narrow": ("bf16", 12, 12, 64, 16, [90, 513, 33], [33, 64, 1], 1, 0, 0.0, "tree"),
    "narrow_e4m3": ("e4m3", 5, 5, 64, 64, [90, 513, 33], [33, 64, 1], 1, 0, 0.0, "tree"),
    "odd_group": ("bf16", 7, 1, 128, 16, [90, 250, 16], [37, 21, 9], 1, 0, 0.0, "tree"),
    "big_group": ("bf16", 24, 1, 64, 128, [190, 250], [64, 50], 1, 0, 0.0, "tree"),
    "big_pages_e4m3": ("e4m3", 6, 2, 64, 256, [1, 255, 256, 257, 1000], [1, 20, 30, 31, 64], 1, 0,
                       0.0, "tree"),
    "more_nodes_than_tokens": ("bf16", 4, 2, 128, 16, [3, 0, 20], [5, 2, 24], 1, 0, 0.0, "tree"),
    "long": ("bf16", 8, 1, 128, 16, [9001], [40], 1, 0, 0.0, "tree"),
    "long_e4m3": ("e4m3", 8, 1, 128, 16, [12007, 50], [25, 25], 1, 0, 0.0, "tree"),
    "long_and_short": ("bf16", 8, 4, 128, 32, [6000, 3, 1, 800, 64], [26, 3, 1, 60, 1], 1, 0, 0.0,
                       "tree"),
    "long_window": ("bf16", 8, 4, 128, 32, [6000, 3, 1, 4000, 64], [26, 3, 1, 60, 1], 1, 2500, 0.0,
                    "tree"),
}

EDGES = {
    "wide_few_e4m3": ("e4m3", 4, 2, 256, 32, [5, 700, 1300, 90], [5, 9, 13, 1], 1, 0, 0.0, "tree"),
    "wide_few_window": ("e4m3", 4, 2, 256, 32, [5, 700, 1300, 90], [5, 9, 13, 1], 1, 333, 50.0, "tree"),
    "wide_one_e4m3": ("e4m3", 3, 3, 256, 16, [1, 17, 33, 520], [1, 1, 1, 1], 1, 0, 0.0, "tree"),
    # more rows than a row block of their average holds
    "wide_ragged_e4m3": ("e4m3", 4, 2, 256, 16, [60, 700, 30, 90, 40], [60, 3, 2, 1, 1], 1, 0, 0.0, "tree"),
    "wide_bits_e4m3": ("e4m3", 2, 2, 256, 16, [33, 64, 300], [9, 30, 17], 1, 0, 0.0, "sparse"),
    # more than a launch's sequences
    "many": ("bf16", 2, 1, 64, 16, [i % 41 for i in range(1030)], [min(i % 3, i % 41) for i in range(1030)],
             1, 0, 0.0, "tree"),
    "far": ("e4m3", 4, 2, 128, 256, [300, 700, 20], [9, 40, 20], 1, 0, 0.0, "tree"),
}


def parents(rng, n, kind="tree"):
    if kind == "chain":
        return list(range(-1, n - 1))
    return [-1] + [int(rng.integers(max(0, i - 7), i)) for i in range(1, n)][:max(n - 1, 0)] if n else []


def trees(rng, new, words, kind):
    """(masks [T, words] uint64, depths [T], parents [T]) of a batch."""
    m, d, par = [], [], []
    for n in new:
        p = parents(rng, n, "chain" if kind == "chain" else "tree")
        a, b = Q.masks(p, words)
        if kind in ("bits", "sparse"):             # any bits, those of later nodes too
            a = rng.integers(0, 2 ** 64, (n, words), dtype=np.uint64)
            if kind == "sparse":
                a &= rng.integers(0, 2 ** 64, (n, words), dtype=np.uint64)
                a[rng.random(n) < 0.4] = 0
        m.append(a)
        d.append(b)
        par += p
    return np.concatenate(m), np.concatenate(d).astype(np.int32), np.array(par, np.int32)


def attend_inputs(name, seed=0):
    cache, Hq, Hkv, D, P, lens, new, words, window, cap, kind = EDGES.get(name) or ATTEND[name]
    rng = np.random.default_rng(len(name) * 1013 + sum(map(ord, name)) + seed)
    table, kv_len, q_start, n = C.batch(rng, lens, new, P)
    K, V, ks, vs = C.dense_pages(rng, n, Hkv, P, D, cache)
    C.poison(K, V, ks, vs, table, lens, P)
    mask, depth, _ = trees(rng, new, words, kind)
    q = f32_to_bf16_bits(rng.normal(0, 2, (int(q_start[-1]), Hq, D)).astype(np.float32))
    return dict(q=q, pages=R.pack(K, V, ks, vs), table=table, kv_len=kv_len, q_start=q_start, P=P,
                D=D, window=window, softcap=cap, new=new, mask=mask, depth=depth)


def widen(x, tokens=4096):
    """A table of that many tokens at least."""
    pad = max(0, tokens // x["P"] - x["table"].shape[1])
    return dict(x, table=np.pad(x["table"], ((0, 0), (0, pad)), constant_values=-1))

"""Tree operators at the edges of their variants: heads of 256 over e4m3 with few rows,
more sequences than a launch takes, pools past 2^32 bytes, graphs that share a
workspace, many moves of a commit."""
from __future__ import annotations

import numpy as np
import pytest

import paged_cases as C
import tree_cases as X
from oracle import paged_ref as R
from oracle import tree_ref as Q
from test_gpu_tree import _attend, _check, _commit, _commit_inputs, _mask

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wide", [0, 16384], ids=["short_table", "long_table"])
@pytest.mark.parametrize("name", [n for n in X.EDGES if n != "far"])
def test_attention(name, wide):
    x = X.widen(X.attend_inputs(name), wide)
    _check(x, _attend(x))


def _far(pages, n):
    """A pool of n pages whose last ones are these."""
    import torch
    pool = torch.empty(n, *pages.shape[1:], dtype=torch.uint8, device="cuda")
    pool[n - pages.shape[0]:] = C.to_gpu(pages)
    return pool


@pytest.mark.parametrize("wide", [0, 16384], ids=["short_table", "long_table"])
def test_attention_past_32_bits(wide):
    import torch
    from chenxing_amd._lib import tree_attention_device
    x = X.widen(X.attend_inputs("far"), wide)
    pages = x["pages"]
    n = (1 << 32) // pages[0].nbytes + 50
    off = n - pages.shape[0]
    pool = _far(pages, n)
    table = np.where(x["table"] >= 0, x["table"] + off, x["table"]).astype(np.int32)
    o = tree_attention_device(C.to_gpu(x["q"]), pool, C.to_gpu(table), C.to_gpu(x["kv_len"]),
                              _mask(x["mask"]), C.to_gpu(x["q_start"]), max_new=max(x["new"]))
    torch.cuda.synchronize()
    _check(x, C.bits_of(o))


def test_commit_past_32_bits():
    """Pages past 2^32 bytes of a layer, and a layer past that."""
    import torch
    from chenxing_amd._lib import kv_commit_device
    _, table, kv_len, q_start, dense, path, count = _commit_inputs("e4m3", 128, 256, 2, 2, [300, 700, 20],
                                                                   [9, 40, 20], 9)
    first = R.pack(*dense[0])
    n = (1 << 32) // first[0].nbytes + 50
    off = n - first.shape[0]
    pool = torch.empty(2, n, *first.shape[1:], dtype=torch.uint8, device="cuda")
    for i, x in enumerate(dense):
        pool[i, off:] = C.to_gpu(R.pack(*x))
    kv_commit_device(pool, 128, C.to_gpu(np.where(table >= 0, table + off, table).astype(np.int32)),
                     C.to_gpu(kv_len), C.to_gpu(path), C.to_gpu(count), C.to_gpu(q_start))
    for i, (K, V, ks, vs) in enumerate(dense):
        Q.commit(K, V, ks, vs, table, kv_len, q_start, path, count, 256)
        assert (C.bits_of(pool[i, off:]) == R.pack(K, V, ks, vs)).all(), i


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("counts", [[140, 65, 40], [33, 64, 32], [32, 31, 37], None])
def test_commit_of_long_paths(cache, counts):
    """Paths of more moves than are looked up at a time; one row stops rising."""
    _, table, kv_len, q_start, dense, _, _ = _commit_inputs(cache, 64, 16, 3, 2, [200, 130, 90],
                                                            [150, 120, 70], 140)
    rng = np.random.default_rng(2)
    path = np.full((3, 140), -1, np.int32)
    for b, (n, k) in enumerate(((150, 140), (120, 65), (70, 40))):
        path[b, :k] = np.sort(rng.choice(n, k, replace=False))
    path[2, 37] = path[2, 36]
    count = None if counts is None else np.array(counts, np.int32)
    _commit(dense, table, kv_len, q_start, path, count, 64, 16)


def test_two_graphs_share_a_workspace():
    import torch
    from chenxing_amd._lib import tree_attention_device
    xs = [X.widen(X.attend_inputs(n, 3)) for n in ("long_and_short", "long_window", "full")]
    ins = [[C.to_gpu(x[k]) for k in ("q", "pages", "table", "kv_len", "q_start", "depth")] +
           [_mask(x["mask"])] for x in xs]

    def call(i):
        a = ins[i]
        return tree_attention_device(a[0], a[1], a[2], a[3], a[6], a[4], a[5], max(xs[i]["new"]),
                                     window=xs[i]["window"])
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for i in range(3):
            call(i)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(call(i))
        graphs.append(g)
    for _ in range(3):
        with torch.cuda.stream(s):
            for o in outs:
                o.zero_()
            for g in graphs:
                g.replay()
            other = call(2)
        torch.cuda.synchronize()
        for x, o in zip(xs, [*outs, other]):
            _check(x, C.bits_of(o))

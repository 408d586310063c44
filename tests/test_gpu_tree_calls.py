"""Calls of the tree operators that their documentation allows at its edges: tables
without columns, paths that stop, windows, scales that vanish."""
from __future__ import annotations

import numpy as np
import pytest

import paged_cases as C
import tree_cases as X
from oracle import paged_ref as R
from oracle import tree_ref as Q
from oracle.bf16 import bf16_bits_to_f32, f32_to_bf16_bits
from test_gpu_tree import _attend, _check, _commit_inputs, _mask

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache,D", [("bf16", 64), ("e4m3", 128), ("e4m3", 256)])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 0, 70]], ids=["one_each", "ragged"])
@pytest.mark.parametrize("window", [0, 5])
def test_tables_without_columns(cache, D, new, window):
    """No slot is held, so every row of a sequence is 0; the rows behind them stay."""
    import torch
    from chenxing_amd._lib import tree_attention_device
    rng = np.random.default_rng(D + sum(new))
    mask, depth, _ = X.trees(rng, new, 2, "tree")
    T = sum(new)
    start = None if max(new) == 1 else C.to_gpu(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
    extra = 0 if start is None else 2
    q = torch.randn(T + extra, 4, D, device="cuda").bfloat16()
    mask = np.concatenate([mask, mask[:extra]])
    depth = np.concatenate([depth, depth[:extra]])
    width = 32 * D if cache == "bf16" else 32 * D + 128
    pool = torch.zeros(3, 2, width, dtype=torch.bfloat16 if cache == "bf16" else torch.uint8, device="cuda")
    out = torch.full_like(q, 7.0)
    tree_attention_device(q, pool, torch.empty(3, 0, dtype=torch.int32, device="cuda"),
                          C.to_gpu(np.array([5, 0, 90], np.int32)), _mask(mask), start, C.to_gpu(depth),
                          max(new), window=window, out=out)
    assert (out[:T] == 0).all() and (out[T:] == 7.0).all()


ROWS = [([0, 4, 2, 8], 2), ([0, 3, 3, 5], 2), ([1, 4, 9, 7], 2), ([-1, 4, 5, 6], 0), ([9, 1, 2, 3], 0),
        ([2, 5, 6, 8], 4), ([0, 4, 8, 1], 3)]


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_paths_that_stop_are_marked(cache):
    """The entry that ends a row before its count becomes -1, for one layer and several;
    a row that ends with its count, or by it, stays as it is."""
    import torch
    from chenxing_amd._lib import kv_commit_device
    B = len(ROWS)
    _, table, kv_len, q_start, dense, _, _ = _commit_inputs(cache, 64, 16, 3, 2, [30] * B, [9] * B, 4)
    path = np.array([r for r, _ in ROWS], np.int32)
    for count in ([4] * B, None, [2] * B):
        for layers in (1, 2):
            pool = torch.stack([C.to_gpu(R.pack(*x)) for x in dense[:layers]])
            p = C.to_gpu(path)
            kv_commit_device(pool, 64, C.to_gpu(table), C.to_gpu(kv_len), p,
                             None if count is None else C.to_gpu(np.array(count, np.int32)),
                             C.to_gpu(q_start))
            want = path.copy()
            for b, (_, n) in enumerate(ROWS):
                if n < (4 if count is None else count[b]):
                    want[b, n] = -1
            assert (p.cpu().numpy() == want).all()


def test_long_paths_that_stop_are_marked():
    """In the second and the third pass of moves."""
    from chenxing_amd._lib import kv_commit_device
    _, table, kv_len, q_start, dense, _, _ = _commit_inputs("bf16", 64, 16, 2, 1, [200] * 4, [150] * 4, 90)
    path = np.tile(np.arange(1, 91, dtype=np.int32), (4, 1))
    for b, at in enumerate((31, 32, 64, 89)):
        path[b, at] = path[b, at - 1]
    p = C.to_gpu(path)
    kv_commit_device(C.to_gpu(R.pack(*dense[0])), 64, C.to_gpu(table), C.to_gpu(kv_len), p,
                     q_start=C.to_gpu(q_start))
    for b, at in enumerate((31, 32, 64, 89)):
        path[b, at] = -1
    assert (p.cpu().numpy() == path).all()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_a_cache_keeps_what_was_moved(cache):
    """PagedKVCache.commit of rows that do not rise: the sequence holds the nodes before
    that, in their order, and nothing behind them."""
    import torch
    from chenxing_amd import PagedKVCache
    c = PagedKVCache(2, 40, 3, 64, 16, dtype=cache)
    seqs = [c.add() for _ in ROWS]
    c.extend(seqs, [21] * len(seqs))
    c.extend(seqs, [9] * len(seqs))
    c.pool.view(torch.uint8).random_(0, 120)
    before = [R.unpack(C.bits_of(x), 64) for x in c.pool]
    batch = c.batch(seqs, [9] * len(seqs))
    path = C.to_gpu(np.array([r for r, _ in ROWS], np.int32))
    count = torch.full((len(seqs),), 4, dtype=torch.int32, device="cuda")
    assert c.commit(seqs, batch, path, count) == [n for _, n in ROWS]
    assert [c.length(s) for s in seqs] == [21 + n for _, n in ROWS]
    for old, x in zip(before, c.pool):
        now = R.unpack(C.bits_of(x), 64)
        for s, (row, n) in zip(seqs, ROWS):
            pages, had = c.pages_of(s), batch["table"][seqs.index(s)].tolist()
            for j in range(n):
                at, frm = 21 + j, 21 + row[j]
                for a, b in zip(now, old):
                    assert (a[pages[at // 16], :, at % 16] == b[had[frm // 16], :, frm % 16]).all()


@pytest.mark.parametrize("new,words,kind", [([1], 1, "tree"), ([64, 65, 0, 63], 2, "tree"), ([130], 1, "chain"),
                                            ([2100, 5], 33, "tree"), ([70, 200], 4, "chain")])
@pytest.mark.parametrize("window", [1, 2, 7, 64, 65, 1 << 30])
def test_masks_of_a_window(new, words, kind, window):
    from chenxing_amd._lib import tree_masks_device
    rng = np.random.default_rng(sum(new) + window % 97)
    par = [X.parents(rng, n, kind) for n in new]
    want = [Q.masks(p, words, window) for p in par]
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    m, d = tree_masks_device(C.to_gpu(np.array(sum(par, []), np.int32)), C.to_gpu(start), words, window)
    assert (m.cpu().numpy().view(np.uint64) == np.concatenate([a for a, _ in want])).all()
    assert (d.cpu().numpy() == np.concatenate([a for _, a in want])).all()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("wide", [0, 4096], ids=["short_table", "long_table"])
@pytest.mark.parametrize("window", [1, 7, 33, 64])
def test_chains_deeper_than_their_window(cache, wide, window):
    """A chain is the causal operator's round, window and all."""
    from chenxing_amd._lib import paged_attention_device, tree_attention_device, tree_masks_device
    X.ATTEND["tmp"] = (cache, 8, 2, 128, 16, [60, 200, 64, 40], [50, 64, 64, 1], 1, window, 0.0, "chain")
    x = X.attend_inputs("tmp", window)
    del X.ATTEND["tmp"]
    x = X.widen(x, wide)
    par = C.to_gpu(np.concatenate([np.arange(-1, n - 1) for n in x["new"]]).astype(np.int32))
    args = [C.to_gpu(x[k]) for k in ("q", "pages", "table", "kv_len")]
    start = C.to_gpu(x["q_start"])
    mask, depth = tree_masks_device(par, start, window=window)
    got = tree_attention_device(*args, mask, start, depth, 64, window=window)
    causal = paged_attention_device(*args, start, 64, window=window)
    K, V = R.unpack(x["pages"], 128)
    want, tol = R.attend(bf16_bits_to_f32(x["q"]).astype(np.float64), K, V, x["table"], x["kv_len"],
                         x["q_start"], 16, 128 ** -0.5, window)
    for o in (got, causal):
        assert (np.abs(bf16_bits_to_f32(C.bits_of(o)) - want) <= tol).all()


@pytest.mark.parametrize("wide", [0, 4096], ids=["short_table", "long_table"])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_scales_below_the_range_of_fp32(wide, softcap):
    """All scores are alike then: a row is the mean of what it attends to."""
    from chenxing_amd._lib import paged_attention_device
    x = X.widen(X.attend_inputs("edges", 4), wide)
    x["softcap"] = softcap
    K, V = R.unpack(x["pages"], x["D"])
    q = bf16_bits_to_f32(x["q"]).astype(np.float64)
    for scale in (1e-46, 1e-60):
        want, tol = Q.attend(q, K, V, x["table"], x["kv_len"], x["q_start"], x["mask"], x["depth"], x["P"],
                             scale, 0, softcap)
        got = bf16_bits_to_f32(_attend(x, scale=scale))
        assert (np.abs(got - want) <= tol).all()
        o = paged_attention_device(C.to_gpu(x["q"]), C.to_gpu(x["pages"]), C.to_gpu(x["table"]),
                                   C.to_gpu(x["kv_len"]), C.to_gpu(x["q_start"]), max(x["new"]),
                                   scale=scale, softcap=softcap)
        want, tol = R.attend(q, K, V, x["table"], x["kv_len"], x["q_start"], x["P"], scale, 0, softcap)
        assert (np.abs(bf16_bits_to_f32(C.bits_of(o)) - want) <= tol).all()


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("wide", [1, 1 << 16], ids=["short_table", "long_table"])
@pytest.mark.parametrize("heads", [2, 40], ids=["few_rows", "many_rows"])
def test_terms_are_not_too_large(cache, D, wide, heads):
    """Terms of 1 and 2^-13 and values of 1 and 33: (1 + 33 2^-13) / (1 + 2^-13) lies 2^-21
    below the middle of 1 and 1 + 2^-7, neighbours in bf16, and goes to 1.  Both sums are
    exact in fp32, the division and the product with it round by 2^-25 and 2^-24: a result
    goes elsewhere only where the terms are more than 2^-22 too large."""
    import torch
    from chenxing_amd._lib import tree_attention_device
    P, nodes = 16, 16
    E = 8 if cache == "bf16" else 16
    ka, va = R._at(P, D, E, 1, np.arange(D))
    _, v0 = R._at(P, D, E, 0, np.arange(D))
    pages = np.zeros((2, 1, 2 * P * D if cache == "bf16" else 2 * P * D + 8 * P),
                     np.uint16 if cache == "bf16" else np.uint8)
    if cache == "bf16":
        bits = f32_to_bf16_bits(np.array([1, 33], np.float32))
        pages[0, 0, ka[0]], pages[0, 0, v0], pages[0, 0, va] = bits[0], bits[0], bits[1]
    else:                                          # codes of 1, and scales
        pages[0, 0, ka[0]] = pages[0, 0, v0] = pages[0, 0, va] = 0x38
        scales = np.ones(2 * P, np.float32)
        scales[P + 1] = 33
        pages[0, 0, 2 * P * D:] = scales.view(np.uint8)
    table = np.full((1, max(2, wide // P)), -1, np.int32)
    table[0, :2] = [0, 1]
    q = torch.zeros(nodes, heads, D, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = -13
    o = tree_attention_device(q, C.to_gpu(pages), C.to_gpu(table),
                              torch.tensor([2 + nodes], dtype=torch.int32, device="cuda"),
                              torch.zeros(nodes, 1, dtype=torch.int64, device="cuda"),
                              torch.tensor([0, nodes], dtype=torch.int32, device="cuda"), max_new=nodes,
                              scale=1 / 1.4426950408889634)
    assert (o == 1).all()


def test_rows_do_not_depend_on_the_workspace():
    """Any contents of the workspace: NaN, ones, another call's; in shares and in chunks."""
    from chenxing_amd import _lib
    for name, wide in (("long_and_short", 0), ("long_and_short", 16384), ("edges_e4m3", 4096), ("full", 0)):
        x = X.widen(X.attend_inputs(name, 12), wide)
        want = _attend(x)
        for byte in (0xFF, 0x7F, 0x01):
            for buf in _lib._ws_tree.bufs.values():
                buf.fill_(byte)
            assert (_attend(x) == want).all(), (name, wide, byte)
        _attend(X.attend_inputs("words"))
        assert (_attend(x) == want).all()


@pytest.mark.parametrize("cache,D", [("bf16", 64), ("e4m3", 128)])
@pytest.mark.parametrize("B,tokens", [(1, 511), (1, 512), (1, 513), (1, 1500), (31, 512), (31, 1500),
                                      (32, 511), (32, 512), (32, 513), (32, 1500), (33, 512), (33, 513),
                                      (64, 200), (65, 200)])
def test_on_both_sides_of_the_chunks(cache, D, B, tokens):
    """256 and 512 workgroups and more, 16 units and more, in tables as long as the longest."""
    rng = np.random.default_rng(B * tokens + D)
    lens = [tokens] + rng.integers(1, tokens, B - 1).tolist()
    new = [int(rng.integers(1, min(n, 5) + 1)) for n in lens]
    X.ATTEND["tmp"] = (cache, 8, 8, D, 16, lens, new, 1, 0, 0.0, "tree")
    x = X.attend_inputs("tmp", B)
    del X.ATTEND["tmp"]
    _check(x, _attend(x))

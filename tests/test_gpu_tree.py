"""Tree attention, masks, accepted paths, commits and appends of drafted trees
against their restatement (oracle/tree_ref.py, oracle/paged_ref.py)."""
from __future__ import annotations

import numpy as np
import pytest

import paged_cases as C
import tree_cases as X
from oracle import paged_ref as R
from oracle import tree_ref as Q
from oracle.bf16 import bf16_bits_to_f32, f32_to_bf16_bits

pytestmark = pytest.mark.gpu


def _values(bits):
    return bf16_bits_to_f32(bits).astype(np.float64)


def _mask(m):
    import torch
    return torch.from_numpy(np.ascontiguousarray(m).view(np.int64)).cuda()


def _attend(x, **kw):
    from chenxing_amd._lib import tree_attention_device
    kw.setdefault("max_new", max([1, *x["new"]]))
    kw.setdefault("depth", C.to_gpu(x["depth"]) if x["window"] else None)
    o = tree_attention_device(C.to_gpu(x["q"]), C.to_gpu(x["pages"]), C.to_gpu(x["table"]),
                              C.to_gpu(x["kv_len"]), _mask(x["mask"]), C.to_gpu(x["q_start"]),
                              window=x["window"], softcap=x["softcap"], **kw)
    return C.bits_of(o)


def _want(x, scale=None):
    K, V = R.unpack(x["pages"], x["D"])
    return Q.attend(_values(x["q"]), K, V, x["table"], x["kv_len"], x["q_start"], x["mask"],
                    x["depth"], x["P"], x["D"] ** -0.5 if scale is None else scale, x["window"],
                    x["softcap"])


def _check(x, got, scale=None):
    want, tol = _want(x, scale)
    got = _values(got)
    off = np.abs(got - want)
    assert np.isfinite(got).all()
    bad = off > tol
    assert not bad.any(), (np.argwhere(bad)[:4].tolist(), float((off / tol).max()))


@pytest.mark.parametrize("name", list(X.ATTEND))
def test_attention(name):
    x = X.attend_inputs(name)
    _check(x, _attend(x))


@pytest.mark.parametrize("name", ["edges", "edges_e4m3", "full", "window", "window_e4m3", "words",
                                  "narrow", "odd_group", "empty_rows", "more_nodes_than_tokens",
                                  "only_nodes", "softcap"])
def test_attention_wide_tables(name):
    """The same in a table that could hold long contexts."""
    x = X.widen(X.attend_inputs(name, 1))
    _check(x, _attend(x))


@pytest.mark.parametrize("hint", [1, 3, 17, 40, 1000])
def test_attention_max_new_is_a_hint(hint):
    x = X.widen(X.attend_inputs("long_and_short", 2))
    _check(x, _attend(x, max_new=hint))


def test_attention_without_q_start():
    import torch
    from chenxing_amd._lib import tree_attention_device
    x = X.attend_inputs("edges")
    x["new"] = [1] * 12
    x["q_start"] = np.arange(13, dtype=np.int32)
    x["mask"], x["q"] = x["mask"][:12] | np.uint64(1), x["q"][:12]
    x["depth"] = np.zeros(12, np.int32)
    o = tree_attention_device(C.to_gpu(x["q"]), C.to_gpu(x["pages"]), C.to_gpu(x["table"]),
                              C.to_gpu(x["kv_len"]), _mask(x["mask"]))
    torch.cuda.synchronize()
    _check(x, C.bits_of(o))


@pytest.mark.parametrize("scale", [1e-3, 0.5])
def test_attention_scale(scale):
    x = X.attend_inputs("chain")
    _check(x, _attend(x, scale=scale), scale)


def test_attention_causal_masks_agree_with_paged_attention():
    """Masks of all earlier nodes are the causal order."""
    from chenxing_amd._lib import paged_attention_device
    x = X.attend_inputs("full", 3)
    for b, n in enumerate(x["new"]):
        r = int(x["q_start"][b])
        for i in range(n):
            x["mask"][r + i, 0] = (1 << (i + 1)) - 1
    _check(x, _attend(x))
    o = paged_attention_device(C.to_gpu(x["q"]), C.to_gpu(x["pages"]), C.to_gpu(x["table"]),
                               C.to_gpu(x["kv_len"]), C.to_gpu(x["q_start"]), max(x["new"]))
    _check(x, C.bits_of(o))


def test_attention_strided_queries():
    import torch
    x = X.attend_inputs("window", 4)
    q = C.to_gpu(x["q"])
    T, H, D = q.shape
    wide = torch.full((T, 2 * H + 1, D + 8), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 1::2][:, :H, :D] = q
    view = wide[:, 1::2][:, :H, :D]
    from chenxing_amd._lib import tree_attention_device
    o = tree_attention_device(view, C.to_gpu(x["pages"]), C.to_gpu(x["table"]),
                              C.to_gpu(x["kv_len"]), _mask(x["mask"]), C.to_gpu(x["q_start"]),
                              C.to_gpu(x["depth"]), max(x["new"]), window=x["window"])
    _check(x, C.bits_of(o))


@pytest.mark.parametrize("widened", [False, True])
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("window", [0, 6])
def test_attention_nan_and_inf_reach_the_rows_that_attend(cache, window, widened):
    """K and V of some nodes and of some tokens at the window's edge are NaN or
    infinite: only rows that attend to them see it."""
    name = "edges" if cache == "bf16" else "edges_e4m3"
    X.ATTEND["tmp"] = (*X.ATTEND[name][:8], window, 0.0, "tree")
    x = X.attend_inputs("tmp", 5)
    del X.ATTEND["tmp"]
    if widened:
        x = X.widen(x)
    P, D = x["P"], x["D"]
    n, H = x["pages"].shape[:2]
    pages = x["pages"].copy()
    E = 8 if cache == "bf16" else 16
    where = {}
    for b, (m, k) in enumerate(zip(x["kv_len"], x["new"])):
        for j, s in enumerate({int(m) - 1, int(m) - k // 2 - 1, max(0, int(m) - k - 3)}):
            pg, o = int(x["table"][b, s // P]), s % P
            ka, va = R._at(P, D, E, o, np.arange(D))
            if cache == "bf16":
                pages[pg, j % H, va[3 + j]] = [0x7FC0, 0x7F80, 0xFF80][j]
            else:
                pages[pg, j % H, va[3 + j]] = 0x7F
            where[(b, s)] = True
    x["pages"] = pages
    K, V = R.unpack(pages, D)
    got = _values(_attend(x))
    G = x["q"].shape[1] // H
    rows = Q.allowed(x["table"], x["kv_len"], x["q_start"], x["mask"], x["depth"], P, n, window)
    clean = dict(x)
    fine = np.isfinite(V)
    want, tol = Q.attend(_values(x["q"]), K, np.where(fine, V, 0.0), x["table"], x["kv_len"],
                         x["q_start"], x["mask"], x["depth"], P, D ** -0.5, window, 0.0)
    del clean
    for t, (b, s) in enumerate(rows):
        pg, o = x["table"][b][s // P], s % P
        for h in range(x["q"].shape[1]):
            v = V[pg, h // G, o]
            with np.errstate(invalid="ignore"):
                special = np.where(np.isfinite(v), 0.0, v).sum(0) if len(s) else np.zeros(D)
            bad = ~np.isfinite(special)
            assert np.isnan(got[t, h][np.isnan(special)]).all(), (t, h)
            inf = np.isinf(special)
            assert (got[t, h][inf] == special[inf]).all(), (t, h)
            assert (np.abs(got[t, h] - want[t, h])[~bad] <= tol[t, h][~bad]).all(), (t, h)


def test_attention_leaves_rows_of_no_sequence():
    import torch
    from chenxing_amd._lib import tree_attention_device
    x = X.attend_inputs("chain", 6)
    T = x["q"].shape[0]
    q = np.concatenate([x["q"], x["q"][:5]])
    mask = np.concatenate([x["mask"], x["mask"][:5]])
    for width in (0, 4096):
        y = X.widen(x, width)
        out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
        tree_attention_device(C.to_gpu(q), C.to_gpu(y["pages"]), C.to_gpu(y["table"]),
                              C.to_gpu(y["kv_len"]), _mask(mask), C.to_gpu(y["q_start"]),
                              max_new=17, out=out)
        assert (out[T:] == 7.0).all()
        _check(x, C.bits_of(out[:T]))


def test_attention_is_the_same_every_time():
    x = X.widen(X.attend_inputs("long_and_short", 7))
    a = _attend(x)
    for _ in range(3):
        assert (_attend(x) == a).all()


def test_attention_captured_and_replayed():
    import torch
    from chenxing_amd._lib import tree_attention_device
    x, y = (X.widen(X.attend_inputs("long_and_short", s)) for s in (8, 9))
    n = max(x["pages"].shape[0], y["pages"].shape[0])
    names = ("q", "pages", "table", "kv_len", "q_start")

    def up(z):
        z = dict(z, pages=np.pad(z["pages"], ((0, n - z["pages"].shape[0]), (0, 0), (0, 0))))
        return [C.to_gpu(z[k]) for k in names] + [_mask(z["mask"])]
    mine = up(x)
    s = torch.cuda.Stream()

    def call():
        return tree_attention_device(mine[0], mine[1], mine[2], mine[3], mine[5], mine[4], max_new=60)
    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for z in (y, x, y):
        for a, b in zip(mine, up(z)):
            a.copy_(b)
        g.replay()
        other = _attend(z)                         # between two replays, on the same stream
        torch.cuda.synchronize()
        _check(z, C.bits_of(out))
        assert (C.bits_of(out) == other).all()


def test_attention_on_two_streams_at_once():
    import torch
    from chenxing_amd._lib import tree_attention_device
    xs = [X.widen(X.attend_inputs("long_and_short", 10)), X.widen(X.attend_inputs("long_window", 11))]
    ins = [[C.to_gpu(x[k]) for k in ("q", "pages", "table", "kv_len", "q_start", "depth")] +
           [_mask(x["mask"])] for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, (x, a, s) in enumerate(zip(xs, ins, streams)):
            with torch.cuda.stream(s):
                outs[i].append(tree_attention_device(a[0], a[1], a[2], a[3], a[6], a[4], a[5], 60,
                                                     window=x["window"]))
    torch.cuda.synchronize()
    for x, o in zip(xs, outs):
        for y in o:
            _check(x, C.bits_of(y))


# ------------------------------------------------------------------ masks, paths
@pytest.mark.parametrize("new,words", [([1], 1), ([0, 3, 0], 1), ([64, 65, 63], 2), ([200, 7], 3),
                                       ([130], 1), ([2100, 5], 33), ([26] * 40, 1)])
def test_masks(new, words):
    from chenxing_amd._lib import tree_masks_device
    rng = np.random.default_rng(sum(new) + words)
    mask, depth, par = X.trees(rng, new, words, "tree")
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    m, d = tree_masks_device(C.to_gpu(par), C.to_gpu(start), words)
    assert (m.cpu().numpy().view(np.uint64) == mask).all()
    assert (d.cpu().numpy() == depth).all()


def test_masks_of_parents_that_are_none():
    """A parent that is not below its node counts as none."""
    from chenxing_amd._lib import tree_masks_device
    par = np.array([-1, 5, 0, 3, 2 ** 31 - 1, -2 ** 31, 2, 6], np.int32)
    m, d = tree_masks_device(C.to_gpu(par), C.to_gpu(np.array([0, 8], np.int32)))
    want, depth = Q.masks(par, 1)
    assert (m.cpu().numpy().view(np.uint64) == want).all() and (d.cpu().numpy() == depth).all()
    m, d = tree_masks_device(C.to_gpu(par))        # eight sequences of one node
    assert (m.cpu().numpy() == 1).all() and (d.cpu().numpy() == 0).all()


@pytest.mark.parametrize("new,width,vocab", [([1], 1, 9), ([0, 3, 0, 1], 4, 2), ([64, 65, 63], 9, 2),
                                             ([300, 7, 256, 257], 12, 3), ([2500], 70, 1),
                                             ([26] * 300, 6, 3), ([90], 1, 1), ([90], 3, 1)])
def test_accept(new, width, vocab):
    from chenxing_amd._lib import tree_accept_device
    rng = np.random.default_rng(sum(new) + width)
    par = np.array([p for n in new for p in X.parents(rng, n)], np.int32)
    start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    tok, out = (rng.integers(0, vocab, len(par)).astype(np.int32) for _ in range(2))
    path, count, nxt = (t.cpu().numpy() for t in tree_accept_device(
        C.to_gpu(par), C.to_gpu(tok), C.to_gpu(out), width, C.to_gpu(start)))
    for b in range(len(new)):
        s = slice(start[b], start[b + 1])
        p, n = Q.accept(par[s], tok[s], out[s], width)
        assert path[b].tolist() == p + [-1] * (width - len(p)) and count[b] == len(p) and nxt[b] == n


# ------------------------------------------------------------------ commit
def _commit_inputs(cache, D, P, H, layers, lens, new, width, seed=0):
    rng = np.random.default_rng(seed + D + P + sum(lens))
    table, kv_len, q_start, n = C.batch(rng, lens, new, P)
    dense = [C.dense_pages(rng, n, H, P, D, cache) for _ in range(layers)]
    path = np.full((len(lens), width), -1, np.int32)
    count = np.zeros(len(lens), np.int32)
    for b, k in enumerate(new):
        c = int(rng.integers(0, min(width, k) + 1))
        path[b, :c] = np.sort(rng.choice(k, c, replace=False)) if c else []
        count[b] = c
    return rng, table, kv_len, q_start, dense, path, count


def _commit(dense, table, kv_len, q_start, path, count, D, P):
    import torch
    from chenxing_amd._lib import kv_commit_device
    pool = torch.stack([C.to_gpu(R.pack(*x)) for x in dense])
    kv_commit_device(pool, D, C.to_gpu(table), C.to_gpu(kv_len), C.to_gpu(path),
                     None if count is None else C.to_gpu(count), C.to_gpu(q_start), page_tokens=P)
    for i, (K, V, ks, vs) in enumerate(dense):
        Q.commit(K, V, ks, vs, table, kv_len, q_start, path, count, P)
        assert (C.bits_of(pool[i]) == R.pack(K, V, ks, vs)).all(), i


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("D,P,H,layers,lens,new,width", [
    (64, 16, 2, 3, [5, 40, 17, 64], [5, 26, 1, 0], 6), (128, 16, 8, 2, [100, 333], [64, 25], 9),
    (256, 32, 3, 1, [70, 31, 33], [64, 31, 32], 20), (128, 128, 1, 4, [300, 129], [64, 64], 64),
    (64, 256, 5, 2, [256, 257, 600], [40, 64, 1], 5), (128, 16, 2, 1, [400], [300], 200)])
def test_commit(cache, D, P, H, layers, lens, new, width):
    _, table, kv_len, q_start, dense, path, count = _commit_inputs(cache, D, P, H, layers, lens, new,
                                                                   width)
    _commit(dense, table, kv_len, q_start, path, count, D, P)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_commit_of_paths_that_stop(cache):
    """Rows that do not rise, reach past the nodes or past the pages, counts past the
    width or below 0, lengths below the nodes."""
    lens, new = [50, 50, 50, 50, 50, 10, 50], [20, 20, 20, 20, 20, 20, 20]
    rng, table, kv_len, q_start, dense, path, count = _commit_inputs(cache, 64, 16, 2, 2, lens, new, 6)
    path[0] = [0, 3, 3, 5, 6, 7]
    path[1] = [2, 1, 5, 6, 7, 8]
    path[2] = [1, 4, 20, 21, 22, 23]
    path[3] = [-1, 4, 5, 6, 7, 8]
    path[4] = path[5] = path[6] = [1, 4, 5, 9, 18, 19]
    count[:] = [6, 6, 6, 6, 600, 6, -3]
    table[4, 3] = -1                               # slots 48 ..: nodes 18 and 19
    _commit(dense, table, kv_len, q_start, path, count, 64, 16)


def test_commit_without_counts_and_of_one_layer():
    from chenxing_amd._lib import kv_commit_device
    _, table, kv_len, q_start, dense, path, count = _commit_inputs("bf16", 128, 16, 2, 1, [90, 40],
                                                                   [33, 20], 7)
    K, V, ks, vs = dense[0]
    page = C.to_gpu(R.pack(K, V))
    kv_commit_device(page, 128, C.to_gpu(table), C.to_gpu(kv_len), C.to_gpu(path),
                     q_start=C.to_gpu(q_start))
    Q.commit(K, V, ks, vs, table, kv_len, q_start, path, None, 16)
    assert (C.bits_of(page) == R.pack(K, V)).all()


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
@pytest.mark.parametrize("many", [False, True])
def test_append_rotates_by_depth(cache, many):
    """A node's q and k as at its depth's position, written to its own slot: the
    result is that of an append of each node alone at that position."""
    from chenxing_amd import rope_table
    from chenxing_amd._lib import kv_append_device
    rng = np.random.default_rng(3)
    D, P, Hq, H = 128, 16, 4, 2
    lens, new = ([50, 33, 70], [20, 33, 1]) if not many else ([300] * 40, [64] * 40)
    table, kv_len, q_start, n = C.batch(rng, lens, new, P)
    _, depth, _ = X.trees(rng, new, 1, "tree")
    T = int(q_start[-1])
    q, k, v = (f32_to_bf16_bits(rng.normal(0, 1, (T, h, D)).astype(np.float32)) for h in (Hq, H, H))
    width = 2 * P * D + (0 if cache == "bf16" else 8 * P)
    kind = np.uint16 if cache == "bf16" else np.uint8
    rope = rope_table(table.shape[1] * P, D)
    pages, plain = (C.to_gpu(np.zeros((n, H, width), kind)) for _ in range(2))
    args = [C.to_gpu(t) for t in (q, k, v)]
    out = kv_append_device(*args, pages, C.to_gpu(table), C.to_gpu(kv_len), C.to_gpu(q_start), rope,
                           depth=C.to_gpu(depth))
    # the rows of rope that the nodes' slots have, replaced by those of their depths
    b = np.repeat(np.arange(len(new)), new)
    i = np.arange(T) - q_start[b]
    base = kv_len[b] - np.array(new)[b]
    for x in range(0, len(new) if not many else 2):
        moved = rope.clone()
        r = slice(int(q_start[x]), int(q_start[x + 1]))
        moved[C.to_gpu((base + i)[r]).long()] = rope[C.to_gpu((base + depth)[r]).long()]
        one = [t[r] for t in args]
        st = np.array([0, new[x]], np.int32)
        o = kv_append_device(*one, plain, C.to_gpu(table[x:x + 1]), C.to_gpu(kv_len[x:x + 1]),
                             C.to_gpu(st), moved)
        assert (C.bits_of(o) == C.bits_of(out[r])).all()
        for pg in table[x][:-(-lens[x] // P)]:
            assert (C.bits_of(pages[int(pg)]) == C.bits_of(plain[int(pg)])).all()


# ------------------------------------------------------------------ a round
def test_a_round_of_trees_together():
    """Trees appended, attended to, walked and committed: the nodes of the accepted
    paths see what a chain of them sees, and the cache goes on, bit for bit, as one
    that appended the accepted tokens alone."""
    from chenxing_amd import PagedKVCache, rope_table, _lib
    rng = np.random.default_rng(11)
    D, P, Hq, H, L = 64, 16, 4, 2, 2
    rope = rope_table(64, D)

    def step(cache, seqs, ids, mask=None, depth=None):
        """Attention outputs of all layers; a token's q, k and v go by its id."""
        new = [len(t) for t in ids]
        cache.extend(seqs, new)
        meta = cache.batch(seqs, new)
        most, table = meta.pop("max_new"), rope[:meta["table"].shape[1] * P]
        outs = []
        for i in range(L):
            x = [np.random.default_rng([int(t), i]).normal(0, 1, (Hq + 2 * H, D)) for s in ids for t in s]
            x = C.to_gpu(f32_to_bf16_bits(np.array(x, np.float32)))
            q = _lib.kv_append_device(x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:], cache.layer(i),
                                      rope=table, depth=depth, **meta)
            if mask is None:
                o = _lib.paged_attention_device(q, cache.layer(i), max_new=most, **meta)
            else:
                o = _lib.tree_attention_device(q, cache.layer(i), mask=mask, max_new=most, **meta)
            outs.append(_values(C.bits_of(o)))
        return outs, meta
    # prompts of 30 and 7 tokens, trees of 13 and 21 nodes whose samples lead to a leaf
    prompts, new = [rng.integers(0, 50, n) for n in (30, 7)], [13, 21]
    par = [X.parents(rng, n) for n in new]
    ids = [np.arange(n) + 100 for n in new]
    sampled, paths, start = np.full(34, 7, np.int32), [], [0, 13, 34]
    for b, n in enumerate(new):
        way = [n - 1]
        while way[0]:
            way.insert(0, par[b][way[0]])
        for a, c in zip(way, way[1:]):
            sampled[start[b] + a] = ids[b][c]
        paths.append(way)
    caches = [PagedKVCache(L, 32, H, D, P) for _ in range(2)]
    seqs = [[c.add(), c.add()] for c in caches]
    for c, s in zip(caches, seqs):
        step(c, s, prompts)
    parents, starts = (C.to_gpu(np.array(x, np.int32)) for x in (sum(par, []), start))
    mask, depth = _lib.tree_masks_device(parents, starts)
    tree, meta = step(caches[0], seqs[0], ids, mask, depth)
    path, count, nxt = _lib.tree_accept_device(
        parents, C.to_gpu(np.concatenate(ids).astype(np.int32)), C.to_gpu(sampled), 12, starts)
    assert [p[:len(w)] for p, w in zip(path.tolist(), paths)] == paths
    assert count.tolist() == [len(w) for w in paths] and nxt.tolist() == [7, 7]
    assert caches[0].commit(seqs[0], meta, path, count) == count.tolist()
    chain, _ = step(caches[1], seqs[1], [t[w] for t, w in zip(ids, paths)])
    for a, b in zip(tree, chain):
        a = np.concatenate([a[s:][w] for s, w in zip(start, paths)])
        # each is off by half a bf16 step and a part in 2^14 of the values' size, about 4
        assert (np.abs(a - b) <= 2 * R.U16 * np.abs(b) + 2.0 ** -12).all()
    assert [caches[0].length(s) for s in seqs[0]] == [caches[1].length(s) for s in seqs[1]]
    for _ in range(2):
        outs = [step(c, s, [[7], [8]])[0] for c, s in zip(caches, seqs)]
        assert (np.array(outs[0]) == np.array(outs[1])).all()

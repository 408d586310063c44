"""PagedKVCache's bookkeeping (CPU: the page copies by torch indexing) against
sequences kept as plain lists, and rope_table against its formula."""
from __future__ import annotations

import math
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from chenxing_amd import OutOfKVCacheError, PagedKVCache, rope_table   # noqa: E402


def _copy(pool, src, dst):
    s, d = src.long(), dst.long()
    assert len(set(d.tolist())) == len(d) and not set(d.tolist()) & set(s.tolist())
    pool[:, d] = pool[:, s]


def _cache(pages=12, **kw):
    return PagedKVCache(2, pages, 1, 64, 16, device="cpu", copy=_copy, **kw)


def _write(c, seq, tokens):
    """Tokens as values at their places, in every layer."""
    pages, n = c.pages_of(seq), c.length(seq)
    for i, t in enumerate(tokens):
        p = n - len(tokens) + i
        c.pool[:, pages[p // 16], 0, p % 16] = float(t)


def _read(c, seq):
    pages = c.pages_of(seq)
    out = [c.pool[:, pages[p // 16], 0, p % 16].tolist() for p in range(c.length(seq))]
    assert all(a == b for a, b in out)
    return [int(a) for a, _ in out]


@pytest.mark.parametrize("seed", range(4))
def test_random_sequences(seed):
    r = random.Random(seed)
    c, want, t = _cache(30), {}, 0
    for _ in range(400):
        op = r.choice(["add", "extend", "extend", "extend", "fork", "truncate", "free", "compact"])
        ids = list(want)
        if op == "add":
            want[c.add()] = []
        elif op == "extend" and ids:
            seqs = r.sample(ids, r.randint(1, min(4, len(ids))))
            counts = [r.choice([0, 1, 1, 2, 17, 33]) for _ in seqs]
            before = {s: (c.pages_of(s), c.length(s)) for s in ids}
            try:
                c.extend(seqs, counts)
            except OutOfKVCacheError:
                assert before == {s: (c.pages_of(s), c.length(s)) for s in ids}
                c.free(ids[0])
                del want[ids[0]]
                continue
            for s, n in zip(seqs, counts):
                new = [(t + i) % 200 for i in range(n)]
                t += n
                _write(c, s, new)
                want[s] += new
        elif op == "fork" and ids:
            s = r.choice(ids)
            for f in c.fork(s, r.randint(1, 3)):
                want[f] = list(want[s])
        elif op == "truncate" and ids:
            s = r.choice(ids)
            n = r.randint(0, len(want[s]))
            c.truncate(s, n)
            want[s] = want[s][:n]
        elif op == "free" and ids:
            s = r.choice(ids)
            c.free(s)
            del want[s]
        elif op == "compact":
            c.compact()
            used = {p for s in want for p in c.pages_of(s)}
            assert used == set(range(len(used)))
        for s, x in want.items():
            assert c.length(s) == len(x) and _read(c, s) == x
        used = {p for s in want for p in c.pages_of(s)}
        assert c.free_pages == 30 - len(used)
    for s in list(want):
        c.free(s)
    assert c.free_pages == 30


def test_sharers_copy_only_what_they_must():
    c = _cache()
    a = c.add()
    c.extend([a], [20])
    b, d = c.fork(a, 2)
    assert c.pages_of(a) == c.pages_of(b) == c.pages_of(d) and c.free_pages == 10
    c.extend([a, b, d], [1, 1, 1])             # the last sharer keeps the page
    assert c.free_pages == 8
    assert len({c.pages_of(s)[1] for s in (a, b, d)}) == 3
    assert len({c.pages_of(s)[0] for s in (a, b, d)}) == 1
    c.extend([a], [11])
    e = c.fork(a)[0]
    c.extend([e], [1])                         # full pages are shared for good
    assert c.pages_of(e)[:2] == c.pages_of(a)


def test_batch():
    c = _cache()
    a, b, e = c.add(), c.add(), c.add()
    c.extend([a, b], [40, 5])
    x = c.batch([b, a, e], [5, 3, 0])
    assert x["table"].tolist() == [[3, -1, -1], [0, 1, 2], [-1, -1, -1]]
    assert x["kv_len"].tolist() == [5, 40, 0] and x["q_start"].tolist() == [0, 5, 8, 8]
    assert x["max_new"] == 5 and x["table"].dtype == torch.int32
    y = c.batch([a])
    assert y["q_start"] is None and y["max_new"] == 1
    assert c.layer(1).shape == (12, 1, 2 * 16 * 64)


def test_refusals():
    for kw in (dict(layers=0), dict(pages=0), dict(kv_heads=0), dict(head_dim=80),
               dict(page_tokens=8), dict(page_tokens=48), dict(dtype="f32")):
        a = dict(layers=1, pages=1, kv_heads=1, head_dim=64, page_tokens=16, dtype="bf16")
        with pytest.raises(ValueError):
            PagedKVCache(**{**a, **kw}, device="cpu")
    c = _cache(2)
    s = c.add()
    for seqs, counts in (([s, s], [1, 1]), ([s], [1, 2]), ([s], [-1])):
        with pytest.raises(ValueError):
            c.extend(seqs, counts)
    with pytest.raises(OutOfKVCacheError):
        c.extend([s], [33])
    c.extend([s], [32])
    with pytest.raises(ValueError):
        c.truncate(s, 33)
    for kw in (dict(positions=-1), dict(rotary_dim=7), dict(theta=0.0), dict(linear=0.0),
               dict(yarn=0.5), dict(original=0)):
        with pytest.raises(ValueError):
            rope_table(**{**dict(positions=4, rotary_dim=8), **kw}, device="cpu")


def test_rope_table():
    t = rope_table(50, 32, 500.0, device="cpu")
    ang = np.arange(50)[:, None] * 500.0 ** (-np.arange(16) / 16)
    want = np.concatenate([np.cos(ang), np.sin(ang)], 1)
    assert t.dtype == torch.float32 and np.abs(t.numpy() - want).max() <= 2.0 ** -24
    assert torch.equal(rope_table(50, 32, 500.0, linear=2.0, device="cpu")[::2], t[:25])
    y = rope_table(9, 64, 10000.0, yarn=4.0, original=2048, device="cpu").double().numpy()
    size = 0.1 * math.log(4) + 1
    ang = np.arange(9)[:, None] * 10000.0 ** (-np.arange(32) / 32)
    # the fastest pair keeps its angle, the slowest turns a quarter as far
    assert np.allclose(y[:, 0], np.cos(ang[:, 0]) * size)
    assert np.allclose(y[:, 31], np.cos(ang[:, 31] / 4) * size)
    assert np.allclose(y[:, :32] ** 2 + y[:, 32:] ** 2, size * size)

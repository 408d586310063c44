"""The tree operators and the 4-bit products refuse bad arguments on the host, before
any device work, and their bindings what their tensors are not (CPU only)."""
from __future__ import annotations

import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from chenxing_amd import _lib, w4                                    # noqa: E402
from oracle import tree_ref as Q                                     # noqa: E402
from oracle import w4_ref as R                                       # noqa: E402
from test_paged_api import A, BAD_BATCH, _kv                         # noqa: E402
from test_workspaces import BF16, I32, _t, device                    # noqa: E402, F401

built = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libcx_sampler.so not built")


def _tree(kv, **kw):
    d = dict(q=A, qt=512, qh=128, heads=4, mask=A, words=1, depth=A, new=1, scale=0.1, window=0,
             cap=0.0, out=A, ws=A, nbytes=1 << 40)
    d.update(kw)
    return _lib.load().cx_tree_attention_bf16(kv, *d.values(), None)


def _commit(kv, **kw):
    d = dict(stride=1 << 20, layers=2, path=A, width=4, count=A)
    d.update(kw)
    return _lib.load().cx_kv_commit(kv, *d.values(), None)


def _append(kv, **kw):
    d = dict(q=A, qt=512, qh=128, k=A, kt=256, kh=128, v=A, vt=256, vh=128, heads=4, rope=A,
             rows=48, rdim=128, inter=0, qn=None, kn=None, eps=1e-6, depth=A, out=A)
    d.update(kw)
    return _lib.load().cx_kv_append_tree_bf16(kv, *d.values(), None)


def _masks(**kw):
    d = dict(parents=A, start=A, B=2, T=9, mask=A, words=1, depth=A)
    d.update(kw)
    return _lib.load().cx_tree_masks(*d.values(), None)


def _accept(**kw):
    d = dict(parents=A, tokens=A, sampled=A, start=A, B=2, T=9, width=4, path=A, count=A, next=A)
    d.update(kw)
    return _lib.load().cx_tree_accept(*d.values(), None)


def _w4(**kw):
    d = dict(x=A, ldx=256, tiles=A, scales=A, shifts=0, group=64, M=2, N=20, K=256, out=A, ldo=20,
             bf16=0)
    d.update(kw)
    return _lib.load().cx_w4_linear_bf16(*d.values(), None)


@built
@pytest.mark.parametrize("bad", BAD_BATCH, ids=str)
def test_bad_batches(bad):
    for call in (_tree, _append):
        assert call(_kv(**bad)) == _lib.CX_EINVAL and _lib.load().cx_last_error()
    if bad != dict(heads=3):                       # (no q heads to divide)
        assert _commit(_kv(**bad)) == _lib.CX_EINVAL
    assert _tree(None) == _commit(None) == _append(None) == _lib.CX_EINVAL


@built
@pytest.mark.parametrize("bad", [
    dict(heads=3), dict(heads=0), dict(mask=0), dict(words=0), dict(words=17), dict(words=-1),
    dict(window=-1), dict(window=5, depth=0), dict(new=0), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e39), dict(cap=-1.0),
    dict(cap=float("nan")), dict(cap=1e-45), dict(scale=1e20, cap=1e-20), dict(q=0), dict(out=0),
    dict(ws=0), dict(q=A + 2), dict(out=A + 8), dict(qt=4), dict(qh=127), dict(ws=A + 8)], ids=str)
def test_bad_tree_attention(bad):
    assert _tree(_kv(), **bad) == _lib.CX_EINVAL and _lib.load().cx_last_error()


@built
def test_tree_attention_workspace():
    size = _lib.load().cx_tree_attention_workspace_bytes
    for D in (64, 128, 256):
        for heads in ((32, 8), (28, 4), (8, 8), (40, 1)):
            last = 0
            for new in [*range(1, 200), 1000, 2 ** 28, 2 ** 31 - 1]:
                n = size(*heads, D, new)
                assert n >= last
                last = n
            need = size(*heads, D, 64)
            if need > 256:
                kv = _kv(D=D, heads=heads[1], T=64, stride=4 * 16 * D * heads[1], M=1 << 20, ld=1 << 20)
                rc = _tree(kv, heads=heads[0], new=64, nbytes=255)
                assert rc == _lib.CX_ENOSPACE


@built
@pytest.mark.parametrize("bad", [dict(stride=-16), dict(stride=8), dict(layers=-1), dict(width=-1),
                                 dict(path=0), dict(layers=2 ** 31 - 1), dict(stride=0)], ids=str)
def test_bad_commits(bad):
    assert _commit(_kv(), **bad) == _lib.CX_EINVAL and _lib.load().cx_last_error()


@built
@pytest.mark.parametrize("bad", [dict(B=-1), dict(T=-1), dict(words=0), dict(parents=0), dict(mask=0),
                                 dict(start=0)], ids=str)
def test_bad_masks(bad):
    assert _masks(**bad) == _lib.CX_EINVAL and _lib.load().cx_last_error()


@built
@pytest.mark.parametrize("bad", [dict(B=-1), dict(T=-1), dict(width=0), dict(parents=0),
                                 dict(tokens=0), dict(sampled=0), dict(path=0), dict(count=0),
                                 dict(next=0), dict(start=0)], ids=str)
def test_bad_accepts(bad):
    assert _accept(**bad) == _lib.CX_EINVAL and _lib.load().cx_last_error()


@built
@pytest.mark.parametrize("bad", [dict(M=-1), dict(N=0), dict(K=0), dict(M=1 << 21), dict(N=1 << 28, ldo=1 << 28),
                                 dict(K=1 << 28, ldx=1 << 28), dict(ldx=255), dict(ldo=19),
                                 dict(group=16), dict(group=0), dict(group=96), dict(K=288, ldx=288),
                                 dict(x=0), dict(tiles=0), dict(scales=0), dict(out=0), dict(x=A + 8),
                                 dict(tiles=A + 4), dict(scales=A + 2), dict(ldx=260), dict(out=A + 2),
                                 dict(out=A + 1, bf16=1)], ids=str)
def test_bad_products(bad):
    assert _w4(**bad) == _lib.CX_EINVAL and _lib.load().cx_last_error()


@built
def test_empty_calls_do_nothing():
    for kw in (dict(B=0, T=0), dict(T=0)):
        assert _tree(_kv(**kw)) == _commit(_kv(**kw)) == _append(_kv(**kw)) == 0
    assert _commit(_kv(), layers=0) == _commit(_kv(), width=0) == 0
    assert _masks(B=0) == _masks(T=0) == _accept(B=0) == _w4(M=0) == 0


# ------------------------------------------------------------------ bindings
def _bad_tensors():
    i32, i64, f32 = I32, torch.int64, torch.float32
    q, cache = _t(6, 4, 64, dtype=BF16), _t(5, 2, 2 * 16 * 64, dtype=BF16)
    table, lens = _t(2, 3, dtype=i32), _t(2, dtype=i32)
    start, mask = _t(3, dtype=i32), _t(6, 1, dtype=i64)

    def tree(**kw):
        d = dict(q=q, cache=cache, table=table, kv_len=lens, mask=mask, q_start=start)
        _lib.tree_attention_device(**{**d, **kw})

    def accept(**kw):
        d = dict(parents=_t(6, dtype=i32), tokens=_t(6, dtype=i32), sampled=_t(6, dtype=i32), width=3,
                 q_start=start)
        _lib.tree_accept_device(**{**d, **kw})

    def commit(**kw):
        d = dict(cache=cache, head_dim=64, table=table, kv_len=lens, path=_t(2, 3, dtype=i32),
                 count=_t(2, dtype=i32), q_start=start)
        _lib.kv_commit_device(**{**d, **kw})

    def product(**kw):
        d = dict(x=_t(3, 256, dtype=BF16), tiles=_t(2, 2, 64, 4, dtype=i32),
                 scales=_t(2, 4, 16, dtype=torch.half), N=20)
        _lib.w4_linear_device(**{**d, **kw})

    def masks(**kw):
        _lib.tree_masks_device(**{**dict(parents=_t(6, dtype=i32), q_start=start), **kw})
    plain = torch.zeros
    return [
        (tree, dict(mask=_t(6, 1, dtype=i32))), (tree, dict(mask=_t(5, 1, dtype=i64))),
        (tree, dict(mask=_t(6, dtype=i64))), (tree, dict(mask=plain(6, 1, dtype=i64))),
        (tree, dict(mask=_t(6, 2, dtype=i64)[:, :1])), (tree, dict(depth=_t(6, dtype=i64))),
        (tree, dict(depth=_t(5, dtype=i32))), (tree, dict(q_start=None)), (tree, dict(q=q.float())),
        (accept, dict(tokens=_t(5, dtype=i32))), (accept, dict(sampled=_t(6, dtype=i64))),
        (accept, dict(parents=_t(6, 1, dtype=i32))), (accept, dict(parents=plain(6, dtype=i32))),
        (accept, dict(tokens=_t(12, dtype=i32)[::2])),
        (masks, dict(parents=_t(6, dtype=i64))), (masks, dict(q_start=_t(3, dtype=i64))),
        (commit, dict(path=_t(3, 3, dtype=i32))), (commit, dict(path=_t(2, dtype=i32))),
        (commit, dict(path=_t(2, 3, dtype=i64))), (commit, dict(count=_t(3, dtype=i32))),
        (commit, dict(head_dim=48)), (commit, dict(page_tokens=32)), (commit, dict(cache=_t(5, 4))),
        (product, dict(x=_t(3, 256))), (product, dict(x=_t(3, 128, dtype=BF16))),
        (product, dict(N=33)), (product, dict(tiles=_t(2, 2, 64, 4))),
        (product, dict(scales=_t(2, 4, 16))), (product, dict(scales=_t(2, 3, 16, dtype=torch.half))),
        (product, dict(scales=_t(2, 4, 16, 3, dtype=torch.half))),
        (product, dict(out=_t(3, 19))), (product, dict(out=_t(3, 20, dtype=torch.half))),
        (product, dict(out=_t(3, 20), dtype=BF16)), (product, dict(out=_t(20, 3).T)),
        (product, dict(dtype=f32, out=_t(3, 20, dtype=BF16))),
    ]


def test_bindings_refuse_other_tensors(device):                          # noqa: F811
    for i, (call, kw) in enumerate(_bad_tensors()):
        with pytest.raises(ValueError):
            call(**kw)
            pytest.fail(f"case {i} was taken")
    assert not device.calls


# ------------------------------------------------------------------ the 4-bit format, the oracle
@pytest.mark.parametrize("N,K,group,shift", [(1, 32, 32, True), (20, 96, 32, False), (16, 128, 128, True),
                                             (50, 448, 64, True), (33, 256, 64, False)])
def test_pack(N, K, group, shift):
    rng = np.random.default_rng(N + K)
    codes = rng.integers(0, 16, (N, K), dtype=np.uint8)
    scale = rng.normal(0, 1, (N, K // group)).astype(np.float16)
    sh = rng.normal(0, 1, scale.shape).astype(np.float16) if shift else None
    args = [None if t is None else torch.from_numpy(t) for t in (codes, scale, sh)]
    tiles, scales = w4.pack(*args)
    want = R.pack(codes, scale, sh)
    assert (tiles.numpy() == want[0]).all() and (scales.numpy() == want[1]).all()
    assert tiles.is_contiguous() and scales.is_contiguous()
    # every code is where the header says
    full = tiles.numpy().view(np.uint32)
    for n, k in zip(rng.integers(0, N, 20), rng.integers(0, K, 20)):
        word = full[n // 16, k // 128, 16 * (k % 32 // 8) + n % 16, k % 128 // 32]
        assert word >> (4 * (k % 8 // 2) + 16 * (k % 2)) & 15 == codes[n, k]


@pytest.mark.parametrize("bad", [dict(codes=torch.zeros(4, 64)), dict(scale=torch.zeros(4, 3)),
                                 dict(scale=torch.zeros(3, 2)), dict(scale=torch.zeros(4, 4)),
                                 dict(shift=torch.zeros(4, 1)),
                                 dict(codes=torch.full((4, 64), 16, dtype=torch.uint8))], ids=str)
def test_pack_refuses(bad):
    d = dict(codes=torch.zeros(4, 64, dtype=torch.uint8), scale=torch.zeros(4, 2), shift=None)
    with pytest.raises(ValueError):
        w4.pack(**{**d, **bad})


def test_quantize_refuses():
    for group in (16, 48, 128):
        with pytest.raises(ValueError):
            w4.quantize(torch.zeros(4, 64), group)
    for bad in (float("nan"), float("inf"), 1e6):
        w = torch.zeros(4, 64)
        w[2, 5] = bad
        with pytest.raises(ValueError):
            w4.quantize(w, 32)


def test_oracle_masks_and_paths():
    m, d = Q.masks([-1, 0, 0, 1, 3, 2], 1)
    assert m[:, 0].tolist() == [1, 3, 5, 11, 27, 37] and d.tolist() == [0, 1, 1, 2, 3, 2]
    assert Q.accept([-1, 0, 0, 1, 2], [5, 6, 7, 8, 9], [7, 0, 9, 0, 4], 9) == ([0, 2, 4], 4)
    assert Q.accept([-1, 0, 0, 1, 2], [5, 6, 7, 8, 9], [7, 0, 9, 0, 4], 2) == ([0, 2], 9)
    assert Q.accept([], [], [], 2) == ([], -1)
    assert Q.moves([0, 2, 4, -1], 3, 5, 10) == [(10, 10), (12, 11), (14, 12)]
    assert Q.moves([0, 2, 2, 4], 4, 5, 10) == [(10, 10), (12, 11)] and Q.moves([0, 1], 2, 5, -1) == []


def test_commit_bookkeeping(monkeypatch):
    """PagedKVCache.commit moves the accepted tokens and lets the rest go."""
    from chenxing_amd import PagedKVCache
    calls = []
    monkeypatch.setattr(_lib, "kv_commit_device", lambda *a: calls.append(a))
    c = PagedKVCache(1, 20, 2, 64, 16, device="cpu")
    seqs = [c.add(), c.add()]
    c.extend(seqs, [15, 40])
    c.extend(seqs, [20, 9])
    batch = c.batch(seqs, [20, 9])
    path, count = torch.zeros(2, 5, dtype=I32), torch.tensor([3, 1], dtype=I32)
    assert c.commit(seqs, batch, path, count) == [3, 1]
    assert [c.length(s) for s in seqs] == [18, 41] and [len(c.pages_of(s)) for s in seqs] == [2, 3]
    assert calls[0][1:] == (64, batch["table"], batch["kv_len"], path, count, batch["q_start"], 16)
    for bad in (torch.tensor([21, 1], dtype=I32), torch.tensor([-1, 1], dtype=I32),
                torch.tensor([1], dtype=I32)):
        with pytest.raises(ValueError):
            c.commit(seqs, batch, path, bad)
    with pytest.raises(ValueError):
        c.commit([seqs[0]] * 2, batch, path, count)
    assert len(calls) == 1


def test_commit_of_a_batch_of_other_lengths_is_refused(monkeypatch):
    from chenxing_amd import PagedKVCache
    calls = []
    monkeypatch.setattr(_lib, "kv_commit_device", lambda *a: calls.append(a))
    c = PagedKVCache(1, 20, 2, 64, 16, device="cpu")
    seqs = [c.add(), c.add()]
    c.extend(seqs, [25, 20])
    batch = c.batch(seqs, [9, 4])
    path, count = torch.tensor([[0, 3], [0, 1]], dtype=I32), torch.tensor([2, 2], dtype=I32)
    with pytest.raises(ValueError):
        c.commit(seqs[::-1], batch, path, count)
    c.extend([seqs[1]], [1])
    with pytest.raises(ValueError):
        c.commit(seqs, batch, path, count)
    c.truncate(seqs[1], 20)
    assert c.commit(seqs, batch, path, count) == [2, 2] and len(calls) == 1
    with pytest.raises(ValueError):            # twice
        c.commit(seqs, batch, path, count)


def test_commit_into_shared_pages_is_refused(monkeypatch):
    """A fork of the appended tree holds the pages that a commit would write to."""
    from chenxing_amd import PagedKVCache
    calls = []
    monkeypatch.setattr(_lib, "kv_commit_device", lambda *a: calls.append(a))
    c = PagedKVCache(1, 20, 2, 64, 16, device="cpu", copy=lambda *a: None)
    s = c.add()
    c.extend([s], [30])
    before, = c.fork(s)                        # shares full pages, and one that extend copies
    c.extend([s], [9])
    batch = c.batch([s], [9])
    path, count = torch.tensor([[0, 3, 8]], dtype=I32), torch.tensor([3], dtype=I32)
    after, = c.fork(s)
    with pytest.raises(ValueError, match="fork"):
        c.commit([s], batch, path, count)
    assert not calls and c.length(s) == 39
    c.commit([s], batch, path, torch.tensor([0], dtype=I32))
    assert c.length(s) == 30
    with pytest.raises(ValueError, match="fork"):
        c.commit([after], batch, path, count)  # slots 30 and 31 are in a page of s
    c.free(s)
    c.free(before)
    assert c.commit([after], batch, path, count) == [3] and c.length(after) == 33

"""Host sides of the tree operators and of the 4-bit products that a call must come
through, on the CPU: no device is looked for or used."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

from chenxing_amd import _lib                                        # noqa: E402
from conftest import ROOT                                            # noqa: E402
from oracle import tree_ref as Q                                     # noqa: E402

built = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libcx_sampler.so not built")

# Calls in a process of their own that sees no device: a launch fails with CX_EHIP.
CALL = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import test_tree_api as T
print(T.{call})
"""


def _alone(call):
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1")
    code = CALL.format(root=ROOT, tests=os.path.join(ROOT, "tests"), call=call)
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])
    return int(r.stdout.split()[-1])


@built
@pytest.mark.parametrize("start", ["", ", q_start=0, T=4"], ids=["q_start", "one_each"])
@pytest.mark.parametrize("window", [0, 5])
def test_a_table_without_columns_is_no_fault(start, window):
    """Every row then attends to nothing: there are no units to divide among workgroups."""
    assert _alone(f"_tree(T._kv(M=0, ld=0, table=0{start}), window={window})") == _lib.CX_EHIP


# ------------------------------------------------------------------ PagedKVCache.commit
@pytest.fixture
def moved(monkeypatch):
    """The calls that commit makes of the device."""
    calls = []
    monkeypatch.setattr(_lib, "kv_commit_device", lambda *a: calls.append(a))
    return calls


def _cache():
    from chenxing_amd import PagedKVCache
    return PagedKVCache(1, 20, 2, 64, 16, device="cpu", copy=lambda *a: None)


def _ids(*rows):
    return torch.tensor(rows, dtype=torch.int32)


def test_commit_after_a_compaction_is_refused(moved):
    """The batch's pages are then another sequence's; a new batch commits."""
    c = _cache()
    a, b = c.add(), c.add()
    c.extend([a, b], [20, 20])
    c.extend([b], [9])
    batch = c.batch([b], [9])
    assert batch["table"].tolist() == [[2, 3]]
    c.free(a)
    c.compact()
    other = c.add()
    c.extend([other], [40])
    assert c.length(b) == 29 and not {2, 3}.isdisjoint(c.pages_of(other))
    path, count = _ids([0, 4, 8]), _ids(3)
    with pytest.raises(ValueError, match="pages"):
        c.commit([b], batch, path, count)
    assert not moved and c.length(b) == 29
    again = c.batch([b], [9])
    assert c.commit([b], again, path, count) == [3] and c.length(b) == 23
    assert moved[0][2].tolist() == [[0, 1]]


def test_commit_after_a_sequence_left_its_pages_is_refused(moved):
    """A fork, an extend and a truncate lead to the same length in a copied page."""
    c = _cache()
    s = c.add()
    c.extend([s], [20])
    c.extend([s], [6])
    batch = c.batch([s], [6])
    c.fork(s)
    c.extend([s], [1])
    c.truncate(s, 26)
    path, count = _ids([0, 4]), _ids(2)
    with pytest.raises(ValueError, match="pages"):
        c.commit([s], batch, path, count)
    assert not moved and c.length(s) == 26
    assert c.commit([s], c.batch([s], [6]), path, count) == [2] and c.length(s) == 22


def test_commit_of_sequences_in_another_order_is_refused(moved):
    c = _cache()
    a, b = c.add(), c.add()
    c.extend([a, b], [30, 30])
    batch = c.batch([a, b], [9, 9])
    path, count = _ids([0, 3], [0, 1]), _ids(2, 2)
    with pytest.raises(ValueError, match="pages"):
        c.commit([b, a], batch, path, count)
    with pytest.raises(ValueError):
        c.commit([a], batch, path, count)
    assert not moved
    assert c.commit([a, b], batch, path, count) == [2, 2] and len(moved) == 1


def test_commit_of_batches_of_single_tokens(moved):
    """Without q_start every sequence has one new token; sequences without pages."""
    c = _cache()
    a, b = c.add(), c.add()
    c.extend([a, b], [17, 1])
    batch = c.batch([a, b])
    assert c.commit([a, b], batch, _ids([0], [-1]), _ids(1, 0)) == [1, 0]
    assert [c.length(a), c.length(b)] == [17, 0] and len(moved) == 1
    empty = c.batch([b], [0])
    assert c.commit([b], empty, _ids([-1]), _ids(0)) == [0] and c.length(b) == 0


def test_commit_of_more_than_the_path_is_refused(moved):
    c = _cache()
    s = c.add()
    c.extend([s], [20])
    c.extend([s], [9])
    batch = c.batch([s], [9])
    with pytest.raises(ValueError, match="count"):
        c.commit([s], batch, _ids([0, 4]), _ids(6))
    for path in (_ids([0, 4], [0, 4]), _ids(0, 4)):
        with pytest.raises(ValueError):
            c.commit([s], batch, path, _ids(2))
    assert not moved and c.length(s) == 29


@pytest.mark.parametrize("row,stays", [([0, 4, 2], 2), ([0, 4, 4], 2), ([0, 4, 9], 2), ([-1, 4, 5], 0),
                                       ([9, 4, 5], 0), ([0, 4, 8], 3)], ids=str)
def test_commit_keeps_what_was_moved(monkeypatch, row, stays):
    """Of a row that stops rising, or passes the nodes, the tokens before that: the
    device call ends there, and marks the place."""
    calls = []

    def device(pool, D, table, kv_len, path, count, *rest):
        calls.append(path.tolist())
        if stays < 3:
            path[1, stays] = -1
    monkeypatch.setattr(_lib, "kv_commit_device", device)
    c = _cache()
    a, b = c.add(), c.add()
    c.extend([a, b], [20, 30])
    batch = c.batch([a, b], [6, 9])
    path = _ids([0, 5, -1], row)
    assert c.commit([a, b], batch, path, _ids(2, 3)) == [2, stays]
    assert len(calls) == 1 and [c.length(a), c.length(b)] == [16, 21 + stays]


# ------------------------------------------------------------------ masks of a window
@built
@pytest.mark.parametrize("bad", [dict(window=-1), dict(B=-1), dict(words=0), dict(parents=0), dict(start=0)],
                         ids=str)
def test_bad_window_masks(bad):
    d = dict(parents=1 << 20, start=1 << 20, B=2, T=9, mask=1 << 20, words=1, depth=1 << 20, window=3)
    d.update(bad)
    assert _lib.load().cx_tree_masks_window(*d.values(), None) == _lib.CX_EINVAL


def test_oracle_window_masks():
    m, d = Q.masks([-1, 0, 0, 1, 3, 2, 4], 1, 3)
    assert m[:, 0].tolist() == [1, 3, 5, 11, 2 + 8 + 16, 1 + 4 + 32, 8 + 16 + 64]
    assert d.tolist() == [0, 1, 1, 2, 3, 2, 4]
    for w in (0, 5, 100):
        assert (Q.masks([-1, 0, 0, 1, 3, 2, 4], 1, w)[0] == Q.masks([-1, 0, 0, 1, 3, 2, 4], 1)[0]).all()
    assert (Q.masks([-1, 0, 1], 1, 1)[0][:, 0] == [1, 2, 4]).all()


# ------------------------------------------------------------------ 4-bit weights
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), 65520.0, -1e30])
@pytest.mark.parametrize("which", ["scale", "shift"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_pack_refuses_what_float16_does_not_hold(value, which, dtype):
    """Scales and shifts are kept as float16: one beyond it would make a row of W infinite."""
    from chenxing_amd import w4
    d = dict(scale=torch.ones(20, 2, dtype=dtype), shift=torch.ones(20, 2, dtype=dtype))
    w4.pack(torch.zeros(20, 64, dtype=torch.uint8), **d)
    d[which][17, 1] = value
    with pytest.raises(ValueError, match="float16"):
        w4.pack(torch.zeros(20, 64, dtype=torch.uint8), **d)


def test_pack_takes_the_largest_of_float16():
    from chenxing_amd import w4
    scale = torch.full((1, 1), -65504.0)
    _, laid = w4.pack(torch.zeros(1, 32, dtype=torch.uint8), scale, -scale)
    assert laid[0, 0, 0].tolist() == [-65504.0, 65504.0]
    # a wider shift is rounded once, not to the scale's type first
    _, laid = w4.pack(torch.zeros(1, 32, dtype=torch.uint8), torch.ones(1, 1, dtype=torch.bfloat16),
                      torch.full((1, 1), 1 + 2.0 ** -9))
    assert laid[0, 0, 0].tolist() == [1.0, 1 + 2.0 ** -9]

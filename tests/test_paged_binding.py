"""What the binding reads of its tensors, or refuses (CPU: host tensors that
pass for device ones, the library replaced)."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")

from chenxing_amd import _lib                                        # noqa: E402
from test_workspaces import BF16, I32, _t, device                    # noqa: E402, F401


def _batch(table, B=3, heads=2, D=64, P=16, cache=None, **kw):
    cache = _t(5, heads, 2 * P * D, dtype=BF16) if cache is None else cache
    block, _ = _lib._kv_batch(torch, 0, cache, D, table, _t(B, dtype=I32), None, B, **kw)
    return dict(zip(("pages", "stride", "table", "ld", "lens", "start", "n", "heads", "D", "P",
                     "dtype", "B", "M", "T"), _lib._KV_BATCH.unpack(block)))


@pytest.mark.parametrize("table,ld", [
    (lambda: _t(3, 4, dtype=I32), 4),
    (lambda: _t(3, 9, dtype=I32)[:, 2:6], 9),
    (lambda: _t(6, 4, dtype=I32)[::2], 8),
    (lambda: _t(3, 1, dtype=I32), 1),
    (lambda: _t(3, 0, dtype=I32), 1),
    (lambda: _t(4, dtype=I32).expand(3, 4)[:1], 4),        # one row: its stride says nothing
    (lambda: _t(9, 1, dtype=I32).as_strided((1, 4), (2, 1)), 4)])
def test_table_rows_are_where_their_stride_says(table, ld):
    t = table()
    x = _batch(t, B=t.shape[0])
    assert (x["ld"], x["M"], x["B"]) == (ld, t.shape[1], t.shape[0])


@pytest.mark.parametrize("table", [
    lambda: _t(4, dtype=I32).expand(3, 4),
    lambda: _t(20, dtype=I32).as_strided((3, 4), (2, 1)),
    lambda: _t(20, dtype=I32).as_strided((3, 4), (3, 1)),
    lambda: _t(4, 3, dtype=I32).T], ids=["expanded", "overlapping", "by one", "transposed"])
def test_tables_whose_rows_overlap_are_refused(table):
    with pytest.raises(ValueError, match="table"):
        _batch(table())


def test_pages_of_another_head_width_are_refused(device):                 # noqa: F811
    """A pool of heads of 128 in pages of 16 has the width of heads of 64 in pages
    of 32: what the cache says of itself has to agree."""
    from chenxing_amd import PagedKVCache
    cache = PagedKVCache(1, 5, 2, 128, 16, device="cpu")
    s = cache.add()
    cache.extend([s], [3])
    x = cache.batch([s])
    most = x.pop("max_new")
    x = {k: v.as_subclass(type(_t(1))) if hasattr(v, "as_subclass") else v for k, v in x.items()}
    pages = cache.layer(0).as_subclass(type(_t(1)))
    for D, fits in ((128, True), (64, False)):
        q, k = _t(1, 4, D, dtype=BF16), _t(1, 2, D, dtype=BF16)
        for call in (lambda: _lib.kv_append_device(q, k, k, pages, **x),
                     lambda: _lib.paged_attention_device(q, pages, max_new=most, **x)):
            if fits:
                call()
            else:
                with pytest.raises(ValueError, match="page of 16 tokens"):
                    call()
    assert len(device.calls) == 2


@pytest.mark.parametrize("theta", [1.0, 0.5])
def test_yarn_needs_angles_that_fall(theta):
    from chenxing_amd import rope_table
    with pytest.raises(ValueError, match="theta"):
        rope_table(4, 8, theta, yarn=2.0, device="cpu")
    assert rope_table(4, 8, theta, device="cpu").shape == (4, 8)

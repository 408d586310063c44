"""Append at the edges of its arguments."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,heads", [(3, 4), (700, 64)])
def test_a_rope_without_rows_is_not_read(T, heads):
    """A table without pages needs no row of the rope: q leaves as it came.  (The
    memory behind the pointer is there, and NaN.)"""
    print(f"[gpu] append, rope without rows, {T} tokens", flush=True)
    import torch
    from chenxing_amd import _lib
    D = 64
    q = torch.randn(T, heads, D, device="cuda").bfloat16()
    k = torch.randn(T, heads, D, device="cuda").bfloat16()
    out = torch.zeros_like(q)
    nan = torch.full((64, D), float("nan"), device="cuda")
    lens = torch.tensor([T], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    pool = torch.zeros(1, heads, 2 * 16 * D, dtype=torch.bfloat16, device="cuda")
    kv = _lib._KV_BATCH.pack(pool.data_ptr(), heads * 2 * 16 * D * 2, 0, 0, lens.data_ptr(),
                             start.data_ptr(), 1, heads, D, 16, _lib.KV_BF16, 1, 0, T)
    row = heads * D
    _lib._check(_lib.load().cx_kv_append_bf16(
        kv, q.data_ptr(), row, D, k.data_ptr(), row, D, k.data_ptr(), row, D, heads, nan.data_ptr(),
        0, D, 0, None, None, 1e-6, out.data_ptr(), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(out, q) and not pool.any()


def test_tokens_without_a_position():
    """New tokens past the table's pages: q is rotated as at position 0, k and v are
    not written."""
    print("[gpu] append past the table", flush=True)
    import torch
    from chenxing_amd._lib import kv_append_device
    D, T = 64, 4
    q, k = (torch.randn(T, 2, D, device="cuda").bfloat16() for _ in range(2))
    pool = torch.zeros(2, 2, 2 * 16 * D, dtype=torch.bfloat16, device="cuda")
    table = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    rope = torch.randn(16, D, device="cuda")
    lens = torch.tensor([17, 2 ** 31 - 1, 0, -5], dtype=torch.int32, device="cuda")
    got = kv_append_device(q, k, k, pool, table, lens, rope=rope)
    one = torch.ones(T, dtype=torch.int32, device="cuda")
    assert not pool.any()
    assert torch.equal(got, kv_append_device(q, k, k, pool, table, one, rope=rope))


def test_a_model_whose_last_position_is_inside_a_page():
    """37 positions in pages of 16: the rope covers whole pages, a shorter one is
    refused."""
    print("[gpu] a rope of 37 positions", flush=True)
    import torch
    from chenxing_amd import PagedKVCache, _lib, rope_table
    T, bf = 37, torch.bfloat16
    cache = PagedKVCache(2, pages=8, kv_heads=8, head_dim=128)
    a = cache.add()
    cache.extend([a], [T])
    batch = cache.batch([a], [T])
    most = batch.pop("max_new")
    q, k, v = (torch.randn(T, h, 128, device="cuda").to(bf) for h in (32, 8, 8))
    rope = rope_table(-(-T // 16) * 16, 128, theta=500000.0)
    with pytest.raises(ValueError, match="positions"):
        _lib.kv_append_device(q, k, v, cache.layer(0), rope=rope[:T], **batch)
    for i in range(2):
        q1 = _lib.kv_append_device(q, k, v, cache.layer(i), rope=rope, **batch)
        o = _lib.paged_attention_device(q1, cache.layer(i), max_new=most, **batch)
    assert torch.equal(o[0], v[0].repeat_interleave(4, 0)) and o.isfinite().all()
    b, = cache.fork(a)
    cache.truncate(a, 20)
    assert (cache.length(a), cache.length(b)) == (20, T)

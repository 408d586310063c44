"""NaN and infinities in V at positions that some of a tile's rows attend to and
others do not, over every head width and tile."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import paged_ref as R
from oracle.bf16 import bf16_bits_to_f32, f32_to_bf16_bits
import paged_cases as C

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("cache,D,G,new,window", [
    ("bf16", 64, 3, 5, 0), ("bf16", 64, 4, 6, 4), ("bf16", 64, 5, 9, 0), ("bf16", 64, 8, 8, 3),
    ("bf16", 128, 2, 4, 0), ("bf16", 128, 3, 9, 0), ("bf16", 128, 5, 9, 5), ("bf16", 256, 3, 9, 0),
    ("e4m3", 64, 2, 6, 0), ("e4m3", 64, 4, 8, 3), ("e4m3", 128, 2, 7, 0), ("e4m3", 256, 3, 9, 4)])
def test_values_that_only_some_rows_attend_to(cache, D, G, new, window, wide):
    print(f"[gpu] attention {cache} heads of {D}, {G} x {new} rows, window {window}, wide {wide}",
          flush=True)
    import torch
    from chenxing_amd._lib import paged_attention_device
    rng = np.random.default_rng(D + G + new)
    P, H, lens = 16, 2, [40, 9, 130, 1000, 64]
    news = [min(new, n) for n in lens]
    table, kv_len, q_start, n = C.batch(rng, lens, news, P, width=4096 // P if wide else None)
    K, V, ks, vs = C.dense_pages(rng, n, H, P, D, cache)
    for b, (length, m) in enumerate(zip(lens, news)):
        for i in range(m):                     # several of the new tokens, in different dims
            pos = length - m + i
            at = rng.choice(D, 3, replace=False)
            V[table[b, pos // P], b % H, pos % P, at[:i % 3]] = \
                C.NAN8 if cache == "e4m3" else [C.NAN16, 0x7F80, 0xFF80][(b + i) % 3]
    C.poison(K, V, ks, vs, table, lens, P)
    q = f32_to_bf16_bits(rng.normal(0, 1, (sum(news), H * G, D)).astype(np.float32))
    pages = R.pack(K, V, ks, vs)
    Kd, Vd = R.unpack(pages, D)
    want, tol = R.attend(bf16_bits_to_f32(q).astype(np.float64), Kd, Vd, table, kv_len, q_start, P,
                         D ** -0.5, window)
    out = paged_attention_device(C.to_gpu(q), C.to_gpu(pages), C.to_gpu(table), C.to_gpu(kv_len),
                                 C.to_gpu(q_start), max_new=new, window=window)
    torch.cuda.synchronize()
    got = bf16_bits_to_f32(C.bits_of(out)).astype(np.float64)
    assert np.isnan(want).any() and np.isfinite(want).mean() > 0.5
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    fine = np.isfinite(want)
    assert (np.abs(got[fine] - want[fine]) <= tol[fine]).all()

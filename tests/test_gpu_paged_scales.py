"""e4m3 rows of every magnitude: without norm and rotation the scale is the fp32
quotient max|x| / 448 and a code the nearest e4m3 value of the fp32 quotient
x / scale, both rounded once, so nothing is left to a tolerance."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import paged_ref as R
from oracle.bf16 import bf16_bits_to_f32, f32_to_bf16_bits
import paged_cases as C

pytestmark = pytest.mark.gpu


def _rows(rng, T, H, D):
    """bf16 bits: every row with a magnitude of its own, from the smallest
    denormal to the largest number, of several smaller ones and zeros."""
    top = rng.integers(-133, 128, (T, H, 1))
    top[:4] = [[[-133]], [[-126]], [[-122]], [[127]]]
    x = rng.uniform(0.5, 1, (T, H, D)) * rng.choice([-1, 1], (T, H, D))
    x = x * 2.0 ** (top - rng.integers(0, 14, (T, H, D)))
    x[rng.random((T, H, D)) < 0.2] = 0.0
    return f32_to_bf16_bits(x.astype(np.float32))


@pytest.mark.parametrize("D,P,H,T", [(64, 16, 2, 300), (128, 16, 3, 300), (256, 32, 1, 300),
                                     (64, 16, 64, 400), (128, 32, 32, 400), (256, 64, 16, 400)])
def test_codes_are_the_quotients(D, P, H, T):
    print(f"[gpu] append e4m3, heads of {D}, {T} tokens of {H} heads", flush=True)
    from chenxing_amd._lib import kv_append_device
    rng = np.random.default_rng(D + H)
    table, kv_len, q_start, n = C.batch(rng, [T], [T], P)
    k, v = (_rows(rng, T, H, D) for _ in range(2))
    q = np.zeros((T, H, D), np.uint16)
    pages = C.to_gpu(np.zeros((n, H, 2 * P * D + 8 * P), np.uint8))
    kv_append_device(C.to_gpu(q), C.to_gpu(k), C.to_gpu(v), pages, C.to_gpu(table),
                     C.to_gpu(kv_len), C.to_gpu(q_start))
    got = C.bits_of(pages)
    sc = np.ascontiguousarray(got[:, :, 2 * P * D:]).view(np.float32)
    d = np.arange(D)
    for t in range(T):
        pg, o = table[0, t // P], t % P
        for bits, at, s in ((k, R._at(P, D, 16, o, d)[0], sc[pg, :, o]),
                            (v, R._at(P, D, 16, o, d)[1], sc[pg, :, P + o])):
            x = bf16_bits_to_f32(bits[t])
            want = np.abs(x).max(1) / np.float32(448)
            want[want == 0] = 1
            assert np.array_equal(s, want), (t, s, want)
            assert np.array_equal(got[pg][:, at], R.e4m3_codes(x / want[:, None])), (t, want)

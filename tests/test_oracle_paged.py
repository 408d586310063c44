"""Pins of the paged cache's 64-bit restatement (oracle/paged_ref.py): the
8-bit format, the page layout, the rotation and attention against direct
formulas."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import paged_ref as R
from oracle.bf16 import bf16_bits_to_f32, f32_to_bf16_bits


def test_e4m3_values_and_codes():
    v = R.E4M3
    assert v[0x7E] == 448 and v[1] == 2.0 ** -9 and v[8] == 2.0 ** -6 and np.isnan(v[[0x7F, 0xFF]]).all()
    fine = ~np.isnan(v)
    codes = np.arange(256)[fine]
    assert np.array_equal(R.e4m3_codes(v[fine]), codes)
    torch = pytest.importorskip("torch")
    x = np.random.default_rng(0).normal(0, 60, 20000).astype(np.float32)
    x = np.concatenate([x, x * 1e-4, (v[:0x7E] + v[1:0x7F]).astype(np.float32) / 2])
    x = x[np.abs(x) <= 448]
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(R.e4m3_codes(x), want)


@pytest.mark.parametrize("P,D", [(16, 64), (32, 128), (256, 256)])
def test_pages_hold_every_element_once(P, D):
    k = np.arange(P * D, dtype=np.uint16).reshape(1, 1, P, D)
    for dt, E in ((np.uint16, 8), (np.uint8, 16)):
        pages = R.pack(k.astype(dt), (k // 7).astype(dt))
        o, d = P - 3, D - 5
        ka = ((d // E) * P + o) * E + d % E
        va = P * D + ((o // E) * D + d) * E + o % E
        assert pages[0, 0, ka] == k[0, 0, o, d].astype(dt)
        assert pages[0, 0, va] == (k[0, 0, o, d] // 7).astype(dt)
    K, V = R.unpack(R.pack(f32_to_bf16_bits(k.astype(np.float32)),
                           f32_to_bf16_bits(-k.astype(np.float32))), D)
    assert np.array_equal(K, bf16_bits_to_f32(f32_to_bf16_bits(k.astype(np.float32))))
    assert np.array_equal(V, -K)


def test_rotation_is_a_product_of_complex_numbers():
    rng = np.random.default_rng(1)
    x = rng.normal(size=(3, 2, 16))
    ang = rng.normal(size=(10, 4))
    rope = np.concatenate([np.cos(ang), np.sin(ang)], 1)
    pos = np.array([0, 7, 3])
    for inter in (False, True):
        y = R.rotate(x, pos, rope, inter)
        a, b = (x[..., 0:8:2], x[..., 1:8:2]) if inter else (x[..., :4], x[..., 4:8])
        z = (a + 1j * b) * np.exp(1j * ang[pos])[:, None]
        ya, yb = (y[..., 0:8:2], y[..., 1:8:2]) if inter else (y[..., :4], y[..., 4:8])
        assert np.allclose(ya, z.real) and np.allclose(yb, z.imag)
        assert np.array_equal(y[..., 8:], x[..., 8:])


@pytest.mark.parametrize("window,softcap", [(0, 0.0), (5, 0.0), (0, 2.0), (3, 1.0)])
def test_attention_is_the_dense_formula(window, softcap):
    rng = np.random.default_rng(2)
    H, G, D, P, n = 2, 3, 16, 4, 6
    K, V = rng.normal(size=(2, n, H, P, D))
    table = np.array([[4, 1, 5], [0, 3, -1]])
    lens, st = [10, 6], [0, 3, 4]
    q = rng.normal(size=(4, H * G, D))
    out, tol = R.attend(q, K, V, table, lens, st, P, 0.3, window, softcap)
    for t, (b, pos) in enumerate([(0, 7), (0, 8), (0, 9), (1, 5)]):
        k = K[table[b]].transpose(1, 0, 2, 3).reshape(H, -1, D)
        v = V[table[b]].transpose(1, 0, 2, 3).reshape(H, -1, D)
        s = np.arange(k.shape[1])
        ok = (s <= pos) & ((s > pos - window) if window else True)
        for h in range(H * G):
            x = 0.3 * k[h // G] @ q[t, h]
            x = softcap * np.tanh(x / softcap) if softcap else x
            p = np.where(ok, np.exp(x), 0)
            assert np.allclose(out[t, h], (p / p.sum()) @ v[h // G])
    assert (tol[out != 0] > 0).all() and (tol < 0.05).all()


def test_attention_of_nothing_is_zero():
    K = np.ones((1, 1, 4, 16))
    out, _ = R.attend(np.ones((3, 1, 16)), K, K, [[0], [0], [-1]], [0, 1, 1], [0, 1, 2, 3], 4, 1.0)
    assert not out[[0, 2]].any() and out[1].all()

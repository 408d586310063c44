"""The paged cache's entry points refuse bad arguments on the host, before any
device work (CPU only), and their argument block has the header's layout."""
from __future__ import annotations

import ctypes as C
import os

import pytest

from chenxing_amd import _lib

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH),
                                reason="libcx_sampler.so not built")
A = 1 << 20                                    # an aligned address that nothing reads


def _kv(**kw):
    d = dict(pages=A, stride=2 * 4096 * 2, table=A, ld=3, lens=A, q_start=A, n=5, heads=2, D=128,
             P=16, dtype=1, B=4, M=3, T=7, **{})
    d.update(kw)
    return _lib._KV_BATCH.pack(*d.values())


def _append(kv, **kw):
    d = dict(q=A, qt=512, qh=128, k=A, kt=256, kh=128, v=A, vt=256, vh=128, heads=4, rope=A,
             rows=48, rdim=128, inter=0, qn=None, kn=None, eps=1e-6, out=A)
    d.update(kw)
    return _lib.load().cx_kv_append_bf16(kv, *d.values(), None)


def _attend(kv, **kw):
    d = dict(q=A, qt=512, qh=128, heads=4, new=1, scale=0.1, window=0, cap=0.0, out=A, ws=A,
             nbytes=1 << 40)
    d.update(kw)
    return _lib.load().cx_paged_attention_bf16(kv, *d.values(), None)


def test_batch_block_layout():
    assert _lib._KV_BATCH.size == 80
    assert _kv(B=0, T=0, pages=0, lens=0) is not None
    # an empty batch is a no-op
    assert _append(_kv(B=0, T=0)) == 0 and _attend(_kv(B=0, T=0)) == 0
    assert _append(_kv(T=0)) == 0 and _attend(_kv(T=0)) == 0


BAD_BATCH = [dict(B=-1), dict(T=-1), dict(n=-1), dict(M=-1), dict(heads=0), dict(ld=2),
             dict(B=4097), dict(D=80), dict(D=0), dict(P=8), dict(P=24), dict(P=512), dict(dtype=0),
             dict(dtype=2), dict(heads=3), dict(q_start=0), dict(stride=2 * 4096 * 2 - 16),
             dict(stride=2 * 4096 * 2 + 8), dict(pages=A + 8), dict(M=1 << 28, ld=1 << 28),
             dict(lens=0), dict(table=0), dict(pages=0),
             dict(dtype=3, stride=2 * (4096 + 128) - 16)]


@pytest.mark.parametrize("bad", BAD_BATCH, ids=str)
def test_bad_batches(bad):
    for call in (_append, _attend):
        assert call(_kv(**bad)) == _lib.CX_EINVAL
        assert _lib.load().cx_last_error()
    assert _append(None) == _attend(None) == _lib.CX_EINVAL


@pytest.mark.parametrize("bad", [
    dict(rdim=24), dict(rdim=8), dict(rdim=144), dict(rows=47), dict(eps=-1e-9),
    dict(eps=float("nan")), dict(q=None), dict(k=None), dict(v=None), dict(out=None),
    dict(q=A + 2), dict(k=A + 8), dict(out=A + 4), dict(qt=516), dict(kh=132), dict(vt=1),
    dict(qn=A + 2), dict(rope=A + 4), dict(heads=3), dict(heads=0)], ids=str)
def test_bad_append_arguments(bad):
    assert _append(_kv(), **bad) == _lib.CX_EINVAL


@pytest.mark.parametrize("bad", [
    dict(new=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(window=-1),
    dict(cap=-1.0), dict(cap=float("nan")), dict(q=None), dict(out=None), dict(ws=None),
    dict(q=A + 2), dict(out=A + 8), dict(qt=4), dict(heads=5)], ids=str)
def test_bad_attention_arguments(bad):
    assert _attend(_kv(), **bad) == _lib.CX_EINVAL


def test_more_work_than_a_call_takes():
    kv = _kv(M=1 << 22, ld=1 << 22, T=1 << 22)
    assert _attend(kv) == _lib.CX_EINVAL and b"too many tokens" in _lib.load().cx_last_error()


def test_attention_workspace():
    lib = _lib.load()
    need = lib.cx_paged_attention_workspace_bytes(4, 2, 128, 1)
    assert need > 0
    assert _attend(_kv(), nbytes=need - 1) == _lib.CX_ENOSPACE
    for bad in ((0, 2, 128, 1), (4, 0, 128, 1), (4, 2, 0, 1), (4, 2, 128, 0)):
        assert lib.cx_paged_attention_workspace_bytes(*bad) > 0


def _copy(**kw):
    d = dict(pages=A, layer=1 << 20, page=8192, bytes=8192, layers=2, n=4, src=A, dst=A, pairs=3)
    d.update(kw)
    return _lib.load().cx_kv_copy_pages(*d.values(), None)


@pytest.mark.parametrize("bad", [
    dict(pairs=-1), dict(layers=-1), dict(n=-1), dict(bytes=-16), dict(bytes=8208),
    dict(bytes=8200), dict(page=8200), dict(layer=8), dict(layer=-16), dict(pages=A + 4),
    dict(pages=None), dict(src=None), dict(dst=None),
    dict(layers=1 << 20, pairs=1 << 20)], ids=str)
def test_bad_copies(bad):
    assert _copy(**bad) == _lib.CX_EINVAL


def test_empty_copies():
    for none in (dict(pairs=0), dict(layers=0), dict(n=0), dict(bytes=0)):
        assert _copy(**none, src=None, dst=None) == 0


def test_cpu_tensors_are_refused():
    torch = pytest.importorskip("torch")
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    cache = torch.zeros(3, 2, 2 * 16 * 64, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        _lib.paged_attention_device(q, cache, i.view(2, 1), i)
    with pytest.raises(ValueError):
        _lib.kv_append_device(q, q[:, :2], q[:, 2:], cache, i.view(2, 1), i)
    with pytest.raises(ValueError):
        _lib.kv_copy_pages_device(cache, i, i)

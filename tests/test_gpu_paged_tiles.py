"""Many sequences of as many rows, more than a tile of heads of 64 holds (the batches
that take four tiles of 16 rows, and those just short of it), and as many sequences as
a call takes."""
from __future__ import annotations

import numpy as np
import pytest

import paged_cases as C
from test_gpu_paged import _attend_torch, _check_many

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,new,G,H,P,window", [
    # 16 tiles in 4 row blocks (6 of three tiles): 98 * 2 * 6 * 22 units, then 92 * ...
    (98, 32, 8, 2, 16, 0), (92, 32, 8, 2, 16, 0), (98, 32, 8, 2, 32, 100),
    # 8 tiles and 7, the last not full
    (200, 16, 8, 2, 16, 0), (200, 21, 5, 2, 16, 50)])
def test_as_many_new_tokens_each(B, new, G, H, P, window):
    print(f"[gpu] attention, {B} sequences of {new} new tokens, {G} heads a kv head", flush=True)
    import torch
    from chenxing_amd._lib import paged_attention_device
    rng = np.random.default_rng(B + new)
    lens = rng.integers(new, 701, B)
    lens[0] = 700
    table, kv_len, q_start, n = C.batch(rng, lens.tolist(), [new] * B, P)
    g = torch.Generator(device="cuda").manual_seed(B)
    K, V = (torch.randn(n, H, P, 64, generator=g, device="cuda").bfloat16() for _ in range(2))
    pages = torch.cat([K.view(n, H, P, 8, 8).transpose(2, 3).reshape(n, H, -1),
                       V.view(n, H, P // 8, 8, 64).transpose(3, 4).reshape(n, H, -1)], 2)
    q = (2 * torch.randn(B * new, G * H, 64, generator=g, device="cuda")).bfloat16()
    out = paged_attention_device(q, pages, C.to_gpu(table), C.to_gpu(kv_len), C.to_gpu(q_start),
                                 max_new=new, window=window).double()
    tab = C.to_gpu(table).long()
    for b in range(B):
        L = int(lens[b])
        pos = torch.arange(L - new, L, device="cuda").repeat_interleave(G)
        rows, pg = slice(b * new, (b + 1) * new), tab[b, :-(-L // P)]
        for h in range(H):
            k, v = (x[pg, h].reshape(-1, 64)[:L].double() for x in (K, V))
            qh, got = (x[rows, h * G:(h + 1) * G].reshape(new * G, 64).double() for x in (q, out))
            want, tol = _attend_torch(qh, k, v, pos, 0.125, window)
            assert ((got - want).abs() <= tol).all(), (b, h, L)


@pytest.mark.parametrize("name,args", [
    ("most_e4m3", ("e4m3", 2, 1, 256, 16, 4096, 0, 40, 2, 0)),
    ("most_singles", ("bf16", 3, 1, 64, 16, 4096, 0, 30, 1, 0))])
def test_the_most_sequences_of_a_call(name, args):
    print(f"[gpu] attention {name}", flush=True)
    _check_many(name, *args)

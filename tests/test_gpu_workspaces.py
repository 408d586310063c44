"""Calls recorded in a HIP graph keep their scratch through later, larger calls, and
threads that share a stream do not share it at once."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _attention(new, pages=512):
    """Two requests of up to 8192 tokens, ``new`` new ones each: the two-launch path."""
    import torch
    from chenxing_amd._lib import paged_attention_device
    g = torch.Generator(device="cuda").manual_seed(new)
    cache = torch.randn(pages, 8, 2 * 16 * 128, generator=g, device="cuda").bfloat16()
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None].repeat(2, 1)
    lens = torch.tensor([7000, 8100], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, new, 2 * new], dtype=torch.int32, device="cuda")
    q = torch.randn(2 * new, 32, 128, generator=g, device="cuda").bfloat16()
    out = torch.zeros_like(q)
    return lambda: paged_attention_device(q, cache, table, lens, start, max_new=new, out=out)


def _lmhead(B):
    import torch
    from chenxing_amd._lib import lmhead_argmax_device
    g = torch.Generator(device="cuda").manual_seed(B)
    h, w = (torch.randn(n, 256, generator=g, device="cuda").bfloat16() for n in (B, 5000))
    ids = torch.zeros(B, dtype=torch.int32, device="cuda")
    return lambda: lmhead_argmax_device(h, w, out_id=ids)[0]


def _sample(B):
    import torch
    from chenxing_amd import _lib
    from chenxing_amd.params import RowParams, pack_rows
    rng = np.random.default_rng(B)
    x = torch.from_numpy(rng.normal(0, 3, (B, 40000)).astype(np.float32)).cuda()
    prm = torch.from_numpy(pack_rows([RowParams(temperature=0.8, top_p=0.95)] * B)
                           .view(np.uint8).copy()).cuda()
    u = torch.from_numpy(rng.random(B)).cuda()
    ids = torch.zeros(B, dtype=torch.int32, device="cuda")
    return lambda: _lib.sample_device(x, prm, u, out_id=ids)[0]


def _verify(B):
    import torch
    from chenxing_amd import _lib
    rng = np.random.default_rng(B)
    t, d = (torch.from_numpy(rng.normal(0, 2, (B, n, 20000)).astype(np.float32)).cuda()
            for n in (5, 4))
    ids = torch.from_numpy(rng.integers(0, 20000, (B, 4)).astype(np.int32)).cuda()
    u = torch.from_numpy(rng.random((B, 5))).cuda()
    T = torch.ones(B, device="cuda")
    outs = [torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(4)]
    return lambda: _lib.spec_verify_device(t, d, ids, u, T, *outs)[1]


@pytest.mark.parametrize("warm", [False, True])
@pytest.mark.parametrize("make,small,large", [(_attention, 1, 5), (_lmhead, 8, 200),
                                              (_sample, 4, 64), (_verify, 2, 16)])
def test_graph_beside_larger_calls(make, small, large, warm):
    print(f"[gpu] graph beside larger calls: {make.__name__}, warm {warm}", flush=True)
    import torch
    step = make(small)
    want = step().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        if warm:
            step()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step()
        more = make(large)
        first = more().clone()
        # tensors in whatever memory that call made free
        others = [torch.full((1 << 20,), i, dtype=torch.int32, device="cuda") for i in range(40)]
    side.synchronize()
    for i in range(3):
        with torch.cuda.stream([side, torch.cuda.current_stream()][i % 2]):
            out.zero_()
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        with torch.cuda.stream(side):
            assert torch.equal(more(), first)
        torch.cuda.synchronize()
        for k, t in enumerate(others):
            assert bool((t == k).all()), k


@pytest.mark.parametrize("makes", [[(_attention, 1), (_attention, 5), (_attention, 2)],
                                   [(_lmhead, 8), (_lmhead, 200)], [(_sample, 4), (_sample, 64)],
                                   [(_verify, 2), (_verify, 16)]])
def test_threads_on_one_stream(makes):
    print(f"[gpu] threads on one stream: {makes[0][0].__name__}", flush=True)
    import threading
    import torch
    steps = [f(n) for f, n in makes]
    want = [s().clone() for s in steps]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        for _ in range(40):
            got = steps[i]().clone()
            if not torch.equal(got, want[i]):
                bad.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(steps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad

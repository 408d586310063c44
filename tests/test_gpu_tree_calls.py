"""Calls of the tree operators that their documentation allows at its edges: tables
without columns."""
from __future__ import annotations

import numpy as np
import pytest

import paged_cases as C
import tree_cases as X
from test_gpu_tree import _mask

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache,D", [("bf16", 64), ("e4m3", 128), ("e4m3", 256)])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 0, 70]], ids=["one_each", "ragged"])
@pytest.mark.parametrize("window", [0, 5])
def test_tables_without_columns(cache, D, new, window):
    """No slot is held, so every row of a sequence is 0; the rows behind them stay."""
    import torch
    from chenxing_amd._lib import tree_attention_device
    rng = np.random.default_rng(D + sum(new))
    mask, depth, _ = X.trees(rng, new, 2, "tree")
    T = sum(new)
    start = None if max(new) == 1 else C.to_gpu(np.concatenate([[0], np.cumsum(new)]).astype(np.int32))
    extra = 0 if start is None else 2
    q = torch.randn(T + extra, 4, D, device="cuda").bfloat16()
    mask = np.concatenate([mask, mask[:extra]])
    depth = np.concatenate([depth, depth[:extra]])
    width = 32 * D if cache == "bf16" else 32 * D + 128
    pool = torch.zeros(3, 2, width, dtype=torch.bfloat16 if cache == "bf16" else torch.uint8, device="cuda")
    out = torch.full_like(q, 7.0)
    tree_attention_device(q, pool, torch.empty(3, 0, dtype=torch.int32, device="cuda"),
                          C.to_gpu(np.array([5, 0, 90], np.int32)), _mask(mask), start, C.to_gpu(depth),
                          max(new), window=window, out=out)
    assert (out[:T] == 0).all() and (out[T:] == 7.0).all()

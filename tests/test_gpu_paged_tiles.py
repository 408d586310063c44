"""Many sequences of more rows than a tile of heads of 64 holds (the batches that
take four tiles of 16 rows, and those just short of it), and as many sequences as a
call takes."""
from __future__ import annotations

import pytest

from test_gpu_paged import _check_many

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,args", [
    # 16 tiles in 4 row blocks (6 of three tiles): 98 * 2 * 6 * 22 units, then 92 * ...
    ("four", ("bf16", 16, 2, 64, 16, 98, 1, 700, 32, 0)),
    ("three", ("bf16", 16, 2, 64, 16, 92, 1, 700, 32, 0)),
    ("four_window", ("bf16", 16, 2, 64, 32, 110, 0, 700, 32, 100)),
    # 8 tiles, 7 of them full
    ("four_eight", ("bf16", 8, 1, 64, 16, 160, 600, 2000, 16, 0))])
def test_attention_of_many_rows(name, args):
    print(f"[gpu] attention {name}", flush=True)
    _check_many(name, *args)


@pytest.mark.parametrize("name,args", [
    ("most_e4m3", ("e4m3", 2, 1, 256, 16, 4096, 0, 40, 2, 0)),
    ("most_singles", ("bf16", 3, 1, 64, 16, 4096, 0, 30, 1, 0))])
def test_the_most_sequences_of_a_call(name, args):
    print(f"[gpu] attention {name}", flush=True)
    _check_many(name, *args)

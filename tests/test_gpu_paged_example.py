"""The paged cache's calls together, as a decoder uses them (examples/paged_decode.py):
prefill, forked samples, decode steps, verify rounds and a compaction give the
hidden states of a recomputation without a cache."""
from __future__ import annotations

import os
import sys

import pytest

pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("cache,bound", [
    # bf16 activations of two layers differ by a few roundings of 2^-8 ...
    ("bf16", 0.03),
    # ... and the 8-bit keys and values by roundings of 2^-4 at most, most of
    # which average out
    ("e4m3", 0.1)])
def test_decoder(cache, bound):
    print(f"[gpu] paged decoder, {cache}", flush=True)
    import paged_decode
    assert paged_decode.main(["--cache", cache]) < bound

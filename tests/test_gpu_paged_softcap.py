"""A cap far above the scores leaves them as they are: the capped score's error goes
with the score, not with the cap."""
from __future__ import annotations

import numpy as np
import pytest

from oracle import paged_ref as R
from test_gpu_paged import _attend, _attend_inputs, _check, _values, _widen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("cap", [1e4, 1e6, 1e30, float("inf")])
@pytest.mark.parametrize("name", ["verify", "long_and_short", "long_e4m3", "wide_heads"])
def test_a_cap_far_above_the_scores(name, cap, wide):
    print(f"[gpu] attention {name}, cap {cap}, wide {wide}", flush=True)
    x = dict(_attend_inputs(name), softcap=0.0)
    K, V = R.unpack(x["pages"], x["D"])
    # c tanh(x / c) is x (1 - (x / c)^2 / 3 ..): at most 2^-24 of x off where |x| < c / 2400
    want, tol = R.attend(_values(x["q"]), K, V, x["table"], x["kv_len"], x["q_start"], x["P"],
                         x["D"] ** -0.5, x["window"], 0.0)
    x["softcap"] = cap
    _check(_attend(_widen(x) if wide else x), want, tol)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("cap", [30.0, 256.0, 257.0, 600.0, 3000.0])
@pytest.mark.parametrize("name", ["verify", "long_e4m3"])
def test_caps_among_large_scores(name, cap, wide):
    print(f"[gpu] attention {name}, cap {cap}, wide {wide}, large scores", flush=True)
    x = dict(_attend_inputs(name), softcap=cap)
    K, V = R.unpack(x["pages"], x["D"])
    want, tol = R.attend(_values(x["q"]), K, V, x["table"], x["kv_len"], x["q_start"], x["P"],
                         9.0, x["window"], cap)
    _check(_attend(_widen(x) if wide else x, scale=9.0), want, tol)


@pytest.mark.parametrize("cap", [0.05, 1.0, 5.0])
def test_caps_below_the_scores(cap):
    print(f"[gpu] attention cap {cap}", flush=True)
    x = dict(_attend_inputs("verify"), softcap=cap)
    K, V = R.unpack(x["pages"], x["D"])
    want, tol = R.attend(_values(x["q"]), K, V, x["table"], x["kv_len"], x["q_start"], x["P"],
                         x["D"] ** -0.5, x["window"], cap)
    _check(_attend(x), want, tol)

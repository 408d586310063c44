"""Host sides of the tree operators and of the 4-bit products that a call must come
through, on the CPU: no device is looked for or used."""
from __future__ import annotations

import os
import subprocess
import sys

import pytest

from chenxing_amd import _lib
from conftest import ROOT

built = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libcx_sampler.so not built")

# Calls in a process of their own that sees no device: a launch fails with CX_EHIP.
CALL = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import test_tree_api as T
print(T.{call})
"""


def _alone(call):
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1")
    code = CALL.format(root=ROOT, tests=os.path.join(ROOT, "tests"), call=call)
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr[-500:])
    return int(r.stdout.split()[-1])


@built
@pytest.mark.parametrize("start", ["", ", q_start=0, T=4"], ids=["q_start", "one_each"])
@pytest.mark.parametrize("window", [0, 5])
def test_a_table_without_columns_is_no_fault(start, window):
    """Every row then attends to nothing: there are no units to divide among workgroups."""
    assert _alone(f"_tree(T._kv(M=0, ld=0, table=0{start}), window={window})") == _lib.CX_EHIP

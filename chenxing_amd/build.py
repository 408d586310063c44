"""Build the gfx950 HIP library ``libcx_sampler.so`` in-tree with hipcc."""
from __future__ import annotations

import os
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libcx_sampler.so")
SOURCES = ["cx_api.hip", "cx_sample.hip", "cx_slow.hip", "cx_verify.hip", "cx_head.hip",
           "cx_kv.hip", "cx_attend.hip", "cx_walk.hip",
           "cx_tree.hip", "cx_w4.hip"]

FLAGS = [
    "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-shared",
    "-ffp-contract=off",                        # numpy never fuses multiply-adds
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    "-Wno-unused-result",
]


def build_hist(verbose: bool = False) -> str:
    """The CPython extension that writes a batch's penalty windows from Python
    lists (csrc/cx_hist.c), compiled with the host C compiler."""
    import sysconfig
    out = os.path.join(HERE, "_cxhist" + sysconfig.get_config_var("EXT_SUFFIX"))
    cmd = [os.environ.get("CC", "gcc"), "-O2", "-shared", "-fPIC", "-Wall",
           "-I", sysconfig.get_paths()["include"], "-o", out + ".tmp",
           os.path.join(CSRC, "cx_hist.c")]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("gcc failed building _cxhist")
    os.replace(out + ".tmp", out)
    return out


def _hipcc(args, verbose: bool) -> None:
    cmd = [os.environ.get("HIPCC", "/opt/rocm/bin/hipcc"), *args]
    if verbose:
        print(" ".join(cmd), flush=True)
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        sys.stderr.write(r.stdout + r.stderr)
        raise RuntimeError("hipcc failed building libcx_sampler.so")


def build(verbose: bool = False) -> str:
    """Every source to an object, several at a time, then the library of them."""
    flags = [f for f in FLAGS if f != "-shared"] + ["-I", os.path.join(ROOT, "include"), "-I", CSRC]
    with tempfile.TemporaryDirectory() as tmp, ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
        objs = [os.path.join(tmp, s + ".o") for s in SOURCES]
        list(pool.map(lambda so: _hipcc([*flags, "-c", os.path.join(CSRC, so[0]), "-o", so[1]],
                                        verbose), zip(SOURCES, objs)))
        _hipcc(["--offload-arch=gfx950", "-fPIC", "-shared", "-o", LIB + ".tmp", *objs], verbose)
    os.replace(LIB + ".tmp", LIB)
    build_hist(verbose)
    return LIB


if __name__ == "__main__":
    print(build(verbose=True))

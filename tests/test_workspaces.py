"""The binding's scratch buffers (CPU: the library replaced by one that notes
which buffer each call is given, and when)."""
from __future__ import annotations

import contextlib
import threading
import time

import pytest

torch = pytest.importorskip("torch")

from chenxing_amd import _lib                                        # noqa: E402

BF16, I32 = torch.bfloat16, torch.int32


class Cuda(torch.Tensor):
    """A host tensor that passes for one on device 0."""
    is_cuda = True

    def get_device(self):
        return 0


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(Cuda)


class Library:
    """Every entry point with a workspace: notes (address, bytes, start, end)."""
    def __init__(self, seconds=0.0):
        self.calls, self.seconds = [], seconds

    def __getattr__(self, name):
        if name.endswith("workspace_bytes"):
            # more for a larger call: by B, or by the most new tokens
            return lambda *a: 4096 * (a[-1] if "attention" in name else a[0])

        def entry(*a):
            ws, nbytes, _ = [getattr(x, "value", x) for x in a[-3:]]
            t = time.perf_counter()
            time.sleep(self.seconds)
            self.calls.append((ws, nbytes, t, time.perf_counter()))
            return 0
        return entry


def _sample(n):
    _lib.sample_device(_t(n, 8), _t(n, 64, dtype=torch.uint8), _t(n, dtype=torch.float64))


def _verify(n):
    _lib.spec_verify_device(_t(n, 3, 8), _t(n, 2, 8), _t(n, 2, dtype=I32),
                            _t(n, 3, dtype=torch.float64), _t(n))


def _lmhead(n):
    _lib.lmhead_argmax_device(_t(n, 128, dtype=BF16), _t(8, 128, dtype=BF16))


def _attention(n):
    _lib.paged_attention_device(_t(1, 4, 64, dtype=BF16), _t(3, 2, 2048, dtype=BF16),
                                _t(1, 2, dtype=I32), _t(1, dtype=I32), max_new=n)


CALLS = {"sample": _sample, "verify": _verify, "lmhead": _lmhead, "attention": _attention}


@pytest.fixture
def device(monkeypatch):
    """The fake library on a device 0 with one stream; .capturing says whether
    that stream records a graph."""
    lib = Library()
    lib.capturing = False
    lib.stream = 7
    monkeypatch.setattr(_lib, "_lib", lib)
    monkeypatch.setattr(_lib, "_stream_ptr", lambda dev: _lib._P(lib.stream))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: lib.stream, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: lib.capturing,
                        raising=False)
    for name in ("_ws_sample", "_ws_verify", "_ws_head", "_ws_attend"):
        monkeypatch.setattr(_lib, name, _lib.Workspace())
    _lib._attention_workspace.cache_clear()
    yield lib
    _lib._attention_workspace.cache_clear()


@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
def test_a_stream_keeps_its_buffer(device, call):
    call(2)
    call(1)
    call(2)
    assert len({a for a, *_ in device.calls}) == 1
    device.stream = 8
    call(2)
    assert device.calls[-1][0] != device.calls[0][0]


@pytest.mark.parametrize("warm", [False, True])
@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
def test_a_graph_shares_no_buffer_with_later_calls(device, call, warm):
    """The address that a graph records is never one that another call is given
    or that a larger call makes the binding let go."""
    kept = []
    if warm:
        call(1)
    device.capturing = True
    real = torch.empty, torch.zeros

    def keep(f):
        def g(*a, **kw):                       # a graph's pool keeps what it captured
            kept.append(f(*a, **kw))
            return kept[-1]
        return g
    torch.empty, torch.zeros = map(keep, real)
    try:
        call(1)
    finally:
        torch.empty, torch.zeros = real
    device.capturing = False
    recorded = device.calls[-1][0]
    assert recorded in {t.data_ptr() for t in kept}
    call(1)
    call(5)
    held = [b.data_ptr() for w in (_lib._ws_sample, _lib._ws_verify, _lib._ws_head, _lib._ws_attend)
            for b in w.bufs.values()]
    assert recorded not in held
    assert recorded not in {a for a, *_ in device.calls[-2:]}


@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
def test_threads_on_one_stream_take_turns(device, call):
    """A call's kernels are launched one after the other: two calls that are
    given one buffer do not overlap."""
    device.seconds = 0.003
    start = threading.Barrier(4)

    def work():
        start.wait()
        for n in (1, 3, 2):
            call(n)
    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    calls = sorted(device.calls, key=lambda c: c[2])
    assert len(calls) == 12
    for a, b in zip(calls, calls[1:]):
        assert a[3] <= b[2] or a[0] != b[0]


@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
def test_a_refused_call_leaves_the_buffer_to_others(device, call):
    class Refused(Exception):
        pass

    def refuse(name):
        def entry(*a):
            raise Refused
        return (lambda *a: 256) if name.endswith("workspace_bytes") else entry
    device.calls, good = [], _lib._lib
    _lib._lib = type("L", (), {"__getattr__": lambda self, name: refuse(name)})()
    try:
        with pytest.raises(Refused):
            call(1)
    finally:
        _lib._lib = good
    t = threading.Thread(target=call, args=(1,))
    t.start()
    t.join(10)
    assert not t.is_alive() and len(device.calls) == 1

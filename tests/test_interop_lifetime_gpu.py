"""Memory shared with torch lives as long as anything over it: views of a
tensor made from torch, torch tensors made of those, recorded graphs."""
from __future__ import annotations

import ctypes as C
import gc
import weakref

import numpy as np
import pytest

from gpu_util import backend
from laya_js_b200 import _lib, interop
from laya_js_b200.host import HostTensor

pytestmark = pytest.mark.gpu


@pytest.fixture()
def b():
    import torch
    be = backend()
    interop.useTorchStream(be)
    yield be
    torch.cuda.synchronize()
    _lib.call("lc_set_stream", 0)


def _lend(b, n=1 << 16):
    """(a backend tensor over a torch tensor that nothing else holds, a weak reference to it, its values)."""
    import torch
    t = torch.arange(n, device="cuda", dtype=torch.float32)
    return interop.fromTorch(b, t), weakref.ref(t), np.arange(n, dtype=np.float32)


def _reuse(n=1 << 16):
    """Tensors of the same size, filled with other values: they get the memory if it was given back."""
    import torch
    junk = [torch.full((n,), -1.0, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    return junk


@pytest.mark.parametrize("view", ["reshape", "transpose", "slice", "split"])
def test_views_keep_the_torch_memory(b, view):
    x, ref, v = _lend(b)
    mid = b.reshape(x, [256, 256])
    y, want = {"reshape": lambda: (b.reshape(x, [256, 256]), v.reshape(256, 256)),
               "transpose": lambda: (b.transpose(mid, [1, 0]), v.reshape(256, 256).T),
               "slice": lambda: (b.slice(x, [100], [900]), v[100:900]),
               "split": lambda: (b.split(x, 4, 0), v.reshape(4, -1))}[view]()
    b.dispose(mid)
    del x
    gc.collect()
    assert ref() is not None
    junk = _reuse()
    assert all(np.array_equal(b.read(t).data, w) for t, w in (zip(y, want) if view == "split" else ((y, want),)))
    for t in y if view == "split" else (y,):
        b.dispose(t)
    del y
    gc.collect()
    assert ref() is None
    del junk


def test_a_lent_tensor_is_given_back_with_its_last_reference(b):
    live = b.stats()["live_tensors"]
    x, ref, _ = _lend(b)
    del x
    gc.collect()
    assert ref() is None and b.stats()["live_tensors"] == live
    x, ref, _ = _lend(b)
    b.dispose(x)  # or before
    assert ref() is None and x.disposed


def test_a_torch_tensor_made_of_one_keeps_it(b):
    import torch
    x, ref, v = _lend(b)
    y = interop.toTorch(b, x)
    z = interop.toTorch(b, b.reshape(interop.fromTorch(b, y), [256, 256]))  # (a view given away, its source collected)
    del x, y
    gc.collect()
    assert ref() is not None
    junk = _reuse()
    assert np.array_equal(z.cpu().numpy(), v.reshape(256, 256))
    del z, junk
    gc.collect()
    b.stats()  # tensors that torch gave back are freed by the next call
    gc.collect()
    b.stats()
    assert ref() is None


def test_a_scope_keeps_what_leaves_it(b):
    x, ref, v = _lend(b)
    y = b.scope(lambda: b.reshape(interop.fromTorch(b, interop.toTorch(b, x)), [2, -1]))
    del x
    gc.collect()
    assert ref() is not None
    junk = _reuse()
    assert np.array_equal(b.read(y).data, v.reshape(2, -1))
    b.dispose(y)
    del junk


def test_a_recorded_graph_keeps_it(b):
    x, ref, v = _lend(b)
    import torch
    torch.cuda.synchronize()
    _lib.call("lc_set_stream", 0)  # (torch's default stream cannot be recorded)
    g = C.c_uint64()
    _lib.call("lc_graph_capture_begin")
    y = b.add(x, x)
    b.dispose(y)
    b.dispose(x)
    del x, y
    _lib.call("lc_graph_capture_end", C.byref(g))
    gc.collect()
    assert ref() is not None
    _lib.call("lc_graph_launch", g.value)
    _lib.call("lc_graph_destroy", g.value)
    gc.collect()
    assert ref() is None


def test_memory_given_back_waits_for_the_stream_it_was_used_on(b):
    """y is made and read on one stream, dropped while the library is on
    another; what the library allocates there next must not take y's memory
    before the read has run."""
    import torch
    n = 1 << 20
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    x = torch.arange(n, device="cuda", dtype=torch.float32)
    torch.cuda.synchronize()
    for _ in range(4):
        with torch.cuda.stream(first):
            interop.useTorchStream(b)
            lent = interop.fromTorch(b, x)
            y = interop.toTorch(b, b.scale(lent, 1.0))
            z = torch.empty_like(x)
            torch.cuda._sleep(20_000_000)  # the read is queued behind some ten milliseconds of waiting
            z.copy_(y)
        with torch.cuda.stream(second):
            interop.useTorchStream(b)
            del y
            others = [b.scale(lent, -2.0) for _ in range(4)]  # of y's size
        torch.cuda.synchronize()
        assert torch.equal(z, x)
        for t in others:
            b.dispose(t)


def test_torch_tensors_dropped_by_another_thread(b):
    """A consumer's thread drops exported tensors while this one calls the
    library: every one is freed, once, and nothing else is."""
    import queue
    import threading

    import torch
    before = b.stats()
    q: queue.Queue = queue.Queue()

    def drop():
        while (t := q.get()) is not None:
            del t
    threads = [threading.Thread(target=drop) for _ in range(3)]
    for t in threads:
        t.start()
    x = interop.fromTorch(b, torch.arange(5000, device="cuda", dtype=torch.float32))
    for i in range(1500):
        y = b.scale(x, 1.0)
        z = interop.toTorch(b, b.scale(y, 2.0))
        q.put(z)
        del z
        b.dispose(y)
    y = b.read(b.scale(x, 3.0)).data
    for t in threads:
        q.put(None)
    for t in threads:
        t.join()
    assert np.array_equal(y, np.arange(5000, dtype=np.float32) * 3)
    b.dispose(x)
    after = b.stats()
    assert after["live_tensors"] == before["live_tensors"] + 1 and after["live_bytes"] == before["live_bytes"] + 20000  # (the one that was read)


def test_tensors_dropped_while_a_graph_is_recorded(b):
    import torch
    torch.cuda.synchronize()
    _lib.call("lc_set_stream", 0)
    x = b.fromHost(HostTensor("f32", (1000,), np.arange(1000, dtype=np.float32)))
    y = interop.toTorch(b, b.scale(x, 2.0))
    before = b.stats()["live_tensors"]
    g = C.c_uint64()
    _lib.call("lc_graph_capture_begin")
    del y
    t = b.add(x, x)
    b.dispose(t)
    assert b.stats()["live_tensors"] == before
    _lib.call("lc_graph_capture_end", C.byref(g))
    assert b.stats()["live_tensors"] == before - 1
    _lib.call("lc_graph_launch", g.value)
    _lib.call("lc_graph_destroy", g.value)
    b.dispose(x)
    b.flush()

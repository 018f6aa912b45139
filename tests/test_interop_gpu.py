"""Zero-copy exchange with torch: every dtype both ways, views, lifetimes and
refusals."""
from __future__ import annotations

import gc

import numpy as np
import pytest

from gpu_util import backend
from laya_js_b200 import _lib, interop
from laya_js_b200._lib import LayaCudaError
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


@pytest.mark.parametrize("dtype", list(interop._NAMES))
@pytest.mark.parametrize("shape", [(), (5,), (3, 0, 2), (2, 3, 4)])
def test_both_ways(b, dtype, shape):
    import torch
    v = (torch.arange(int(np.prod(shape))) % 2).reshape(shape).to(getattr(torch, interop._NAMES[dtype])).cuda()
    t = interop.fromTorch(b, v)
    assert t.shape == tuple(shape) and t.dtype == dtype
    back = interop.toTorch(b, b.cast(t, dtype))
    assert back.dtype == v.dtype and back.shape == v.shape and torch.equal(back, v)


def test_memory_is_shared_and_freed_with_the_torch_tensor(b):
    import torch
    before = b.stats()
    y = interop.toTorch(b, b.fromHost(HostTensor("f32", (4, 5), np.arange(20, dtype=np.float32))))
    assert b.stats()["live_tensors"] == before["live_tensors"] + 1
    view = y[1:3]
    del y
    gc.collect()
    assert b.stats()["live_tensors"] == before["live_tensors"] + 1  # the view keeps the memory
    assert view.cpu().tolist() == [[5, 6, 7, 8, 9], [10, 11, 12, 13, 14]]
    del view
    gc.collect()
    assert b.stats() == {**before, "launches": b.stats()["launches"]}
    x = torch.ones(3, device="cuda")
    t = interop.fromTorch(b, x)
    x += 1
    assert b.read(t).data.tolist() == [2, 2, 2]


def test_a_scope_does_not_free_what_torch_holds(b):
    import torch
    got = []
    b.scope(lambda: got.append(interop.toTorch(b, b.fromHost(HostTensor("f16", (3,), np.ones(3, np.float16))))))
    torch.cuda.synchronize()
    assert got[0].cpu().tolist() == [1, 1, 1]


def test_views_and_refusals(b):
    import torch
    t = b.fromHost(HostTensor("f32", (2, 3), np.arange(6, dtype=np.float32)))
    tr = interop.toTorch(b, b.transpose(t, [1, 0]))
    assert tr.cpu().tolist() == [[0, 3], [1, 4], [2, 5]]
    given = b.cast(t, "f32")
    interop.toTorch(b, given)
    with pytest.raises(LayaCudaError, match="dispose"):
        interop.toTorch(b, given)
    with pytest.raises(ValueError, match="contiguous"):
        interop.fromTorch(b, torch.zeros(3, 4, device="cuda").t())
    with pytest.raises(ValueError, match="cpu"):
        interop.fromTorch(b, torch.zeros(3))
    with pytest.raises(TypeError, match="complex"):
        interop.fromTorch(b, torch.zeros(3, dtype=torch.complex64, device="cuda"))

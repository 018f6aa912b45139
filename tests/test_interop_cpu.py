"""The exchange with torch, without a GPU: what the library is asked for, and
what is kept until it answers."""
from __future__ import annotations

import gc
import types
import weakref

import pytest
import torch

from laya_js_b200 import _lib, interop


class _Cuda(torch.Tensor):
    """A CPU tensor that says it is on the device."""

    @property
    def device(self):
        return torch.device("cuda", 0)


@pytest.fixture()
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(_lib, "call", lambda name, *a: made.append((name, a)))
    monkeypatch.setattr(interop, "_torch_stream", lambda device: 1, raising=False)
    return made


def _backend():
    return types.SimpleNamespace(device=0, _scopes=[], dispose=lambda t: None, _destroyed=False,
                                 _wrap=lambda h, dtype, shape: types.SimpleNamespace(handle=h, dtype=dtype, shape=shape))


def test_the_torch_tensor_outlives_the_handle_it_was_made_into(calls):
    """Views share the library's storage, not the Python object: only the
    storage knows when the memory is no longer read."""
    t = torch.zeros(4, 3).as_subclass(_Cuda)
    ref = weakref.ref(t)
    x = interop.fromTorch(_backend(), t)
    assert x.dtype == "f32" and x.shape == (4, 3)
    del t, x
    gc.collect()
    assert ref() is not None
    (name, args), = calls
    assert name == "lc_from_device_owned"
    interop._returned(args[-1], 1)  # as the library does when the last view is gone
    gc.collect()
    assert ref() is None


def test_a_refused_tensor_is_not_kept(monkeypatch, calls):
    def refuse(name, *a):
        raise _lib.LayaCudaError("no")
    monkeypatch.setattr(_lib, "call", refuse)
    t = torch.zeros(4).as_subclass(_Cuda)
    ref = weakref.ref(t)
    with pytest.raises(_lib.LayaCudaError):
        interop.fromTorch(_backend(), t)
    del t
    gc.collect()
    assert ref() is None


def test_tensors_that_would_lose_something_are_refused(calls):
    """Autograd would be cut without a word; a negated view's memory holds the
    other sign."""
    t = torch.zeros(4, requires_grad=True).as_subclass(_Cuda)
    with pytest.raises(ValueError, match="requires grad"):
        interop.fromTorch(_backend(), t)
    with torch.no_grad():
        interop.fromTorch(_backend(), t)
    interop.fromTorch(_backend(), t.detach())
    neg = torch._neg_view(torch.ones(4)).as_subclass(_Cuda)
    with pytest.raises(ValueError, match="negated"):
        interop.fromTorch(_backend(), neg)


def test_a_strided_view_is_known_by_asking(monkeypatch):
    """Not by the words of an error message: any other refusal is passed on."""
    asked = []

    def call(name, *a):
        asked.append(name)
        if name == "lc_tensor_to_dlpack":
            raise _lib.LayaCudaError("the device is dense with errors")
        a[1]._obj.value = 64  # lc_tensor_data: a dense tensor's address
    monkeypatch.setattr(_lib, "call", call)
    b = types.SimpleNamespace(device=0, _h=lambda t, what: t.handle, cast=lambda *a: pytest.fail("copied a dense tensor"))
    t = types.SimpleNamespace(handle=5, disposed=False, dtype="f32")
    with pytest.raises(_lib.LayaCudaError, match="device"):
        interop.toTorch(b, t)
    assert asked == ["lc_tensor_to_dlpack", "lc_tensor_data"]

"""Zero-copy exchange with torch on the backend's device, for programs whose
training loop or data lives in torch.

    useTorchStream(b)            # run the backend's ops on torch's current stream
    x = fromTorch(b, t)          # a CudaTensor over t's memory
    t = toTorch(b, y)            # a torch tensor over y's memory, which it now owns

Both directions share memory: the backend treats tensors as immutable, so a
tensor handed over is read, not written, while a queued op may still use it.
The memory lives as long as anything over it: views of ``x`` (and their
torch tensors) keep ``t``'s, views of ``t`` (and tensors made of it) ``y``'s.
"""
from __future__ import annotations

import ctypes as C
import itertools

from . import _lib
from .backend import CudaTensor, _i64
from .host import CODE

_NAMES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16", "i32": "int32", "bool": "bool", "u8": "uint8", "i8": "int8",
          "i16": "int16", "i64": "int64", "f64": "float64"}
_DTYPES: dict = {}  # torch dtype -> backend dtype, filled on first use
_LEGACY_STREAM = 1  # cudaStreamLegacy: torch's default stream has handle 0, which lc_set_stream takes for the library's own


def _torch_stream(device: int) -> int:
    import torch
    return torch._C._cuda_getCurrentRawStream(device) or _LEGACY_STREAM


def useTorchStream(b) -> None:
    """Makes torch's current stream the library's, so that ops and torch
    kernels run in the order they are issued."""
    _lib.call("lc_set_stream", _torch_stream(b.device))


_lent: dict = {}  # owner -> (torch tensor whose memory the library reads, the torch stream it came from)
_owners = itertools.count(1)


@C.CFUNCTYPE(None, C.c_void_p, C.c_uint64)
def _returned(owner, stream):
    """The library holds no tensor over the memory any more; ops queued on ``stream`` may still read it."""
    t, origin = _lent.pop(owner)
    if stream != origin and t.numel():
        import torch
        if stream == _LEGACY_STREAM:
            t.record_stream(torch.cuda.default_stream(t.device))
        else:
            t.record_stream(torch.cuda.ExternalStream(stream, t.device))


_on_release = C.cast(_returned, C.c_void_p)


class LentTensor(CudaTensor):
    """A tensor over torch's memory. It is disposed when nothing refers to it
    any more, so that a program that only hands torch tensors in has nothing to
    give back; views of it are disposed as any other tensor."""

    __slots__ = ()

    def __del__(self):
        try:
            self._backend.dispose(self)
        except Exception:
            pass  # the library may be gone at interpreter exit


def fromTorch(b, t) -> CudaTensor:
    """A tensor over the memory of ``t`` (contiguous, on the backend's
    device), which stays alive as long as the result, a view of it that was not
    disposed or a recorded graph that reads it."""
    import torch
    if not _DTYPES:
        _DTYPES.update({getattr(torch, v): k for k, v in _NAMES.items()})
    dtype = _DTYPES.get(t.dtype)
    if dtype is None:
        raise TypeError(f"fromTorch: no backend dtype for {t.dtype}")
    if t.device.type != "cuda" or (t.device.index or 0) != b.device:
        raise ValueError(f"fromTorch: tensor on {t.device}, backend on cuda:{b.device}")
    if not t.is_contiguous():
        raise ValueError("fromTorch: the tensor must be contiguous")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError("fromTorch: the tensor requires grad, which the backend's ops do not record; pass t.detach() (or use torch.no_grad())")
    if t.is_neg():
        raise ValueError("fromTorch: the tensor is a negated view; pass t.resolve_neg()")
    out, owner = C.c_uint64(), next(_owners)
    _lent[owner] = (t, _torch_stream(b.device))
    try:
        _lib.call("lc_from_device_owned", C.byref(out), CODE[dtype], _i64(t.shape), t.dim(), t.data_ptr(), _on_release, owner)
    except BaseException:
        del _lent[owner]
        raise
    r = LentTensor(b, out.value, dtype, tuple(t.shape))
    if b._scopes:
        b._scopes[-1].append(r)
    return r


_capsule = C.pythonapi.PyCapsule_New
_capsule.restype, _capsule.argtypes = C.py_object, [C.c_void_p, C.c_char_p, C.c_void_p]


def _is_dense(t: CudaTensor) -> bool:
    p = C.c_uint64()
    _lib.call("lc_tensor_data", t.handle, C.byref(p))
    return p.value != 0


def toTorch(b, t: CudaTensor):
    """``t`` as a torch tensor over the same memory (DLPack). The handle now
    belongs to the torch tensor, which frees it in the order of the library's
    stream, and is not used further; a strided view is copied first."""
    import torch
    out = C.c_uint64()
    try:
        _lib.call("lc_tensor_to_dlpack", b._h(t, "toTorch"), C.byref(out))
    except _lib.LayaCudaError:
        if t.disposed or _is_dense(t):
            raise
        d = b.cast(t, t.dtype)
        b.dispose(t)
        return toTorch(b, d)
    t.disposed = True
    return torch.from_dlpack(_capsule(out.value, b"dltensor", None))

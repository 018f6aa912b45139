"""Zero-copy exchange with torch on the backend's device, for programs whose
training loop or data lives in torch.

    useTorchStream(b)            # run the backend's ops on torch's current stream
    x = fromTorch(b, t)          # a CudaTensor over t's memory
    t = toTorch(b, y)            # a torch tensor over y's memory, which it now owns

Both directions share memory: the backend treats tensors as immutable, so a
tensor handed over is read, not written, while a queued op may still use it.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from .backend import CudaTensor, _i64
from .host import CODE

_NAMES = {"f32": "float32", "f16": "float16", "bf16": "bfloat16", "i32": "int32", "bool": "bool", "u8": "uint8", "i8": "int8",
          "i16": "int16", "i64": "int64", "f64": "float64"}
_LEGACY_STREAM = 1  # cudaStreamLegacy: torch's default stream has handle 0, which lc_set_stream takes for the library's own


def useTorchStream(b) -> None:
    """Makes torch's current stream the library's, so that ops and torch
    kernels run in the order they are issued."""
    import torch
    s = torch.cuda.current_stream(b.device).cuda_stream or _LEGACY_STREAM
    _lib.call("lc_set_stream", s)


def fromTorch(b, t) -> CudaTensor:
    """A tensor over the memory of ``t`` (contiguous, on the backend's
    device), which stays alive as long as the result does."""
    dtype = {v: k for k, v in _NAMES.items()}.get(str(t.dtype).replace("torch.", ""))
    if dtype is None:
        raise TypeError(f"fromTorch: no backend dtype for {t.dtype}")
    if t.device.type != "cuda" or (t.device.index or 0) != b.device:
        raise ValueError(f"fromTorch: tensor on {t.device}, backend on cuda:{b.device}")
    if not t.is_contiguous():
        raise ValueError("fromTorch: the tensor must be contiguous")
    out = C.c_uint64()
    _lib.call("lc_from_device", C.byref(out), CODE[dtype], _i64(t.shape), t.dim(), t.data_ptr())
    r = b._wrap(out.value)
    r.keep = t
    return r


class _Owner:
    """Device memory of a tensor as torch reads it; disposes the tensor when torch lets go."""

    def __init__(self, b, t, ptr, typestr):
        self.b, self.t = b, t
        self.__cuda_array_interface__ = {"shape": t.shape, "typestr": typestr, "data": (ptr, False), "version": 2, "strides": None}

    def __del__(self):
        try:
            self.b.dispose(self.t)
        except Exception:
            pass  # the library may be gone at interpreter exit


_TYPESTR = {"f32": "<f4", "f16": "<f2", "bf16": "<i2", "i32": "<i4", "bool": "|b1", "u8": "|u1", "i8": "|i1", "i16": "<i2", "i64": "<i8",
            "f64": "<f8"}


def toTorch(b, t: CudaTensor):
    """``t`` as a torch tensor over the same memory. The handle now belongs to
    the torch tensor (it is disposed with it, in the order of the library's
    stream) and is not used further."""
    import torch
    if t.dtype not in _TYPESTR:
        raise TypeError(f"toTorch: no torch dtype for {t.dtype}")
    if 0 in t.shape:
        out = torch.empty(t.shape, dtype=getattr(torch, _NAMES[t.dtype]), device=f"cuda:{b.device}")
        b.dispose(t)
        return out
    ptr = C.c_uint64()
    _lib.call("lc_tensor_data", b._h(t, "toTorch"), C.byref(ptr))
    if not ptr.value:
        d = b.cast(t, t.dtype)  # a dense copy of the strided view
        b.dispose(t)
        return toTorch(b, d)
    if b._scopes and any(x is t for x in b._scopes[-1]):
        b._scopes[-1] = [x for x in b._scopes[-1] if x is not t]  # no longer the scope's to dispose
    out = torch.as_tensor(_Owner(b, t, ptr.value, _TYPESTR[t.dtype]), device=f"cuda:{b.device}")
    return out.view(torch.bfloat16) if t.dtype == "bf16" else out

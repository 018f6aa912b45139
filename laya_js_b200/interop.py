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
from math import prod

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
    _lib.call("lc_set_stream", torch._C._cuda_getCurrentRawStream(b.device) or _LEGACY_STREAM)


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

    __slots__ = ("b", "t", "__cuda_array_interface__")

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


class _Owners:
    """Memory that several handles share, as torch reads it; frees those given to torch when torch lets go."""

    __slots__ = ("b", "taken", "__cuda_array_interface__")

    def __init__(self, b, count, ptr, typestr):
        self.b, self.taken = b, []
        self.__cuda_array_interface__ = {"shape": (count,), "typestr": typestr, "data": (ptr, False), "version": 2, "strides": None}

    def __del__(self):
        try:
            if self.taken and not self.b._destroyed:
                _lib.call("lc_tensors_free", (C.c_uint64 * len(self.taken))(*self.taken), len(self.taken))
        except Exception:
            pass  # the library may be gone at interpreter exit


class SharedMemory:
    """Dense tensors that an op returned in one allocation (each one's ``keep``
    is (this, its index)): torch gets views of one storage over it."""

    __slots__ = ("b", "ts", "ptrs", "flat")

    def __init__(self, b, ts):
        self.b, self.ts, self.ptrs, self.flat = b, [(t.handle, t.dtype, t.shape) for t in ts], None, {}
        for i, t in enumerate(ts):
            t.keep = (self, i)

    def _flat(self, dtype: str):
        """(a flat torch tensor from the first to the last tensor of a dtype, its owner's list, address, value size)."""
        import torch
        size = int(_TYPESTR[dtype][-1])
        mine = [(p, prod(sh) * size) for p, (_, dt, sh) in zip(self.ptrs, self.ts) if dt == dtype and 0 not in sh]
        lo, hi = min(p for p, _ in mine), max(p + n for p, n in mine)
        owner = _Owners(self.b, (hi - lo) // size, lo, _TYPESTR[dtype])
        flat = torch.as_tensor(owner, device=f"cuda:{self.b.device}")
        return flat.view(torch.bfloat16) if dtype == "bf16" else flat, owner.taken, lo, size

    def torch(self, t: CudaTensor, i: int):
        if self.ptrs is None:
            n = len(self.ts)
            ptrs = (C.c_uint64 * n)()
            _lib.call("lc_tensors_data", (C.c_uint64 * n)(*[h for h, _, _ in self.ts]), n, ptrs)
            self.ptrs = list(ptrs)
        if t.dtype not in self.flat:
            self.flat[t.dtype] = self._flat(t.dtype)
        flat, taken, lo, size = self.flat[t.dtype]
        strides, s = [], 1
        for d in reversed(t.shape):
            strides.append(s)
            s *= d
        taken.append(t.handle)
        t.disposed = True  # the handle is torch's now
        return flat.as_strided(t.shape, strides[::-1], (self.ptrs[i] - lo) // size)


def toTorch(b, t: CudaTensor):
    """``t`` as a torch tensor over the same memory. The handle now belongs to
    the torch tensor (it is disposed with it, in the order of the library's
    stream) and is not used further."""
    import torch
    if t.dtype not in _TYPESTR:
        raise TypeError(f"toTorch: no torch dtype for {t.dtype}")
    if type(t.keep) is tuple and not t.disposed and 0 not in t.shape:
        return t.keep[0].torch(t, t.keep[1])
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
    for frame in b._scopes:  # no longer a scope's to dispose
        frame[:] = [x for x in frame if x is not t]
    out = torch.as_tensor(_Owner(b, t, ptr.value, _TYPESTR[t.dtype]), device=f"cuda:{b.device}")
    return out.view(torch.bfloat16) if t.dtype == "bf16" else out

"""Low-rank adapters of many requests beside a shared projection, their
gradients, and gradient clipping (include/laya_cuda_adapters.h).

    plan = AdapterPlan(b, cu_rows, adapters, n_adapters)   # once per batch
    y = adapter_linear(b, x, w, bias, a, bt, scales, plan)
    dx, da, db = adapter_linear_grad(b, dy, x, w, a, bt, scales, plan)
    (da, db), norm = clip_grad_norm(b, [da, db], 1.0)

Tensors are the backend's (``CudaTensor``); ``a`` [n, r, in] and ``bt``
[n, r, out] hold the adapters of all tenants, ``bt`` the transpose of the
usual [out, r] matrix (``AdapterBank`` does the layout from host arrays).
``EncoderAdapters`` puts banks beside the projections of a ``ModernBert``:

    tenants = EncoderAdapters(banks).batch([3, -1, 0], length)   # adapter of each prompt
    hidden = model.forward(ids, mask, 3, length, tenants=tenants)
"""
from __future__ import annotations

import ctypes as C
from typing import Sequence

import numpy as np

from . import _lib
from . import compose as Cm
from .host import HostTensor, f32_to_bf16_bits


def _int32(what: str, v) -> np.ndarray:
    v = np.asarray(v)
    if v.size and v.dtype.kind not in "iu":
        raise TypeError(f"AdapterPlan: {what} must be whole numbers, got {v.dtype}")
    if v.size and (v.max() > np.iinfo(np.int32).max or v.min() < np.iinfo(np.int32).min):
        raise ValueError(f"AdapterPlan: {what} must fit 32 bits")
    return np.ascontiguousarray(v, np.int32)


class AdapterPlan:
    """The rows of one batch: request i owns rows cu_rows[i]:cu_rows[i + 1] and
    uses adapter ``adapters[i]`` (-1: none). One plan serves every layer."""

    def __init__(self, backend, cu_rows, adapters, n_adapters: int):
        cu, ad = _int32("cu_rows", cu_rows), _int32("adapters", adapters)
        if cu.ndim != 1 or ad.ndim != 1 or len(cu) != len(ad) + 1:
            raise ValueError(f"AdapterPlan: cu_rows has {cu.shape} entries, adapters {ad.shape}: one more than the requests is expected")
        h = C.c_uint64()
        p32 = C.POINTER(C.c_int32)
        _lib.call("lc_adapter_plan_create", C.byref(h), cu.ctypes.data_as(p32), ad.ctypes.data_as(p32), len(ad), int(n_adapters))
        self.backend, self.handle = backend, h.value
        self.rows, self.n_adapters = int(cu[-1]), int(n_adapters)

    def free(self) -> None:
        if self.handle and not self.backend._destroyed:
            _lib.call("lc_adapter_plan_free", self.handle)
        self.handle = 0

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass  # the library may be gone at interpreter exit


def adapter_linear(backend, x, w, bias, a, bt, scales, plan: AdapterPlan):
    """y = x·wᵀ (+ bias) + s·(x·Aᵀ)·B for each row's adapter; ``w`` None: the
    adapters' share alone (beside a projection that is computed elsewhere)."""
    b, out = backend, C.c_uint64()
    _lib.call("lc_adapter_linear", C.byref(out), b._h(x, "adapter_linear"), b._h(w), b._h(bias), b._h(a), b._h(bt), b._h(scales), plan.handle)
    return b._wrap(out.value, x.dtype, (*x.shape[:-1], bt.shape[2]))


def adapter_linear_grad(backend, dy, x, w, a, bt, scales, plan: AdapterPlan, want: Sequence[str] = ("dx", "da", "db")):
    """(dx, da, db) of adapter_linear for ``dy``; those not in ``want`` are None."""
    unknown = set(want) - {"dx", "da", "db"}
    if unknown:
        raise ValueError(f"adapter_linear_grad: unknown gradients {sorted(unknown)}")
    b = backend
    outs = [C.c_uint64() if k in want else None for k in ("dx", "da", "db")]
    _lib.call("lc_adapter_linear_grad", *[None if o is None else C.byref(o) for o in outs], b._h(dy, "adapter_linear_grad"), b._h(x), b._h(w),
              b._h(a), b._h(bt), b._h(scales), plan.handle)
    return tuple(None if o is None else b._wrap(o.value, x.dtype, like.shape) for o, like in zip(outs, (x, a, bt)))


def clip_grad_norm(backend, grads: Sequence, max_norm: float):
    """(clipped tensors, global norm as an f32 scalar tensor)."""
    b, n = backend, len(grads)
    hs = (C.c_uint64 * max(1, n))(*[b._h(g, "clip_grad_norm") for g in grads])
    outs = (C.c_uint64 * max(1, n))()
    norm = C.c_uint64()
    _lib.call("lc_clip_grad_norm", outs, C.byref(norm), hs, n, float(max_norm))
    return [b._wrap(h, g.dtype, g.shape) for h, g in zip(outs, grads)], b._wrap(norm.value, "f32", ())


def _host(dtype: str, v) -> HostTensor:
    v = np.ascontiguousarray(v, np.float32)
    data = v.astype(np.float16) if dtype == "f16" else f32_to_bf16_bits(v) if dtype == "bf16" else v
    return HostTensor(dtype, v.shape, data)


class AdapterBank:
    """The adapters of all tenants for one projection on the device: from host
    arrays down [n, r, in], up [n, out, r] (the usual orientation) and scales
    [n] (alpha / rank)."""

    def __init__(self, backend, down, up, scales, dtype: str):
        down, up = np.asarray(down, np.float32), np.asarray(up, np.float32)
        scales = np.asarray(scales, np.float32)
        if down.ndim != 3 or up.ndim != 3 or down.shape[0] != up.shape[0] or down.shape[1] != up.shape[2] or scales.shape != down.shape[:1]:
            raise ValueError(f"AdapterBank: down {down.shape}, up {up.shape}, scales {scales.shape}; [n, r, in], [n, out, r] and [n] expected")
        self.backend = backend
        self.a = backend.fromHost(_host(dtype, down))
        self.bt = backend.fromHost(_host(dtype, up.transpose(0, 2, 1)))
        self.scales = backend.fromHost(HostTensor("f32", scales.shape, scales))

    def linear(self, x, w, bias, plan: AdapterPlan):
        return adapter_linear(self.backend, x, w, bias, self.a, self.bt, self.scales, plan)

    def linear_grad(self, dy, x, w, plan: AdapterPlan, want: Sequence[str] = ("dx", "da", "db")):
        return adapter_linear_grad(self.backend, dy, x, w, self.a, self.bt, self.scales, plan, want)

    def dispose(self) -> None:
        for t in (self.a, self.bt, self.scales):
            self.backend.dispose(t)


PROJECTIONS = ("Wqkv", "Wo", "Wi", "WoMlp")


class EncoderAdapters:
    """Adapters beside a ModernBert's projections: per layer a dict from
    projection (``PROJECTIONS``) to its ``AdapterBank``; projections left out
    have none. Every bank holds the same number of tenants."""

    def __init__(self, banks: Sequence[dict]):
        sizes = {bank.a.shape[0] for layer in banks for bank in layer.values()}
        unknown = {name for layer in banks for name in layer} - set(PROJECTIONS)
        if unknown:
            raise ValueError(f"EncoderAdapters: unknown projections {sorted(unknown)}, expected {PROJECTIONS}")
        if len(sizes) != 1:
            raise ValueError(f"EncoderAdapters: every bank must hold the same number of tenants, got {sorted(sizes)}")
        self.banks = list(banks)
        self.n = sizes.pop()
        self.backend = next(bank for layer in banks for bank in layer.values()).backend

    def batch(self, tenants: Sequence[int], length: int) -> "TenantBatch":
        """The adapter of each prompt (-1: none) of a padded batch of ``length`` tokens per prompt."""
        return TenantBatch(self, tenants, length)

    def dispose(self) -> None:
        for layer in self.banks:
            for bank in layer.values():
                bank.dispose()


class TenantBatch:
    """The adapters of one batch of prompts, for ``ModernBert.forward``."""

    def __init__(self, adapters: EncoderAdapters, tenants: Sequence[int], length: int):
        self.adapters = adapters
        cu = np.arange(len(tenants) + 1, dtype=np.int64) * int(length)
        if cu[-1] > np.iinfo(np.int32).max:
            raise ValueError(f"TenantBatch: {cu[-1]} rows are too many")
        self.plan = AdapterPlan(adapters.backend, cu, tenants, adapters.n)

    def linear(self, layer: int, name: str, x, w, bias):
        """The projection ``name`` of a layer with its adapters; a packed weight is multiplied on its own path and the
        adapters' share added."""
        b = self.adapters.backend
        bank = self.adapters.banks[layer].get(name) if layer < len(self.adapters.banks) else None
        if bank is None:
            return Cm.linearAny(b, x, w, bias)
        if Cm.is_quantized(w):
            return b.add(Cm.linearAny(b, x, w, bias), bank.linear(x, None, None, self.plan))
        return bank.linear(x, w, bias, self.plan)

    def free(self) -> None:
        self.plan.free()

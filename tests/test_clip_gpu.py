"""Global-norm gradient clipping against 64 bits: mixed dtypes, sizes around
the kernels' chunks, unaligned and strided gradients, more tensors than one
launch takes, magnitudes whose squares leave f32, non-finite gradients."""
from __future__ import annotations

import math

import numpy as np
import pytest

from adapters_ref import DIGITS, TINY, mk, vals
from gpu_util import backend
from laya_js_b200 import adapters as A
from laya_js_b200._lib import LayaCudaError
from laya_js_b200.host import HostTensor

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _clip(hosts, max_norm):
    b = backend()
    outs, norm = A.clip_grad_norm(b, [b.fromHost(h) for h in hosts], max_norm)
    assert norm.shape == () and norm.dtype == "f32"
    for o, h in zip(outs, hosts):
        assert o.shape == tuple(h.shape) and o.dtype == h.dtype
    return [vals(b.read(o)) for o in outs], float(vals(b.read(norm)))


def _want(hosts, max_norm):
    v = [vals(h) for h in hosts]
    norm = math.sqrt(sum(float(np.sum(x * x)) for x in v))
    f = min(1.0, max_norm / (norm + EPS))
    return [x * f for x in v], norm


def _check(hosts, max_norm):
    """norm: one rounding to f32 of a sum of f64 (or of f32 squares within
    groups of at most 32: 2^-19 in all); values: the factor's and the
    product's f32 roundings and the norm's error, then the dtype's."""
    got, norm = _clip(hosts, max_norm)
    want, n = _want(hosts, max_norm)
    assert abs(norm - n) <= 2.0 ** -19 * n + 1e-45
    for g, w, h in zip(got, want, hosts):
        assert np.all(np.abs(g - w) <= (2.0 ** -DIGITS[h.dtype] + 2.0 ** -18) * np.abs(w) + TINY[h.dtype])


@pytest.mark.parametrize("max_norm", [0.5, 1e9, 0.0, math.inf])
@pytest.mark.parametrize("sizes", [[1], [7], [8191, 8192, 8193], [0, 5, 0], [100000, 3, 65536, 1000003], [2048] * 50])
def test_clip_matches_64_bits(sizes, max_norm):
    rng = np.random.default_rng(sum(sizes))
    kinds = ("f32", "f16", "bf16")
    _check([mk(kinds[i % 3], rng.standard_normal(n) * 10.0 ** rng.uniform(-2, 0)) for i, n in enumerate(sizes)], max_norm)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_shapes_scalars_and_many_tensors(dtype):
    rng = np.random.default_rng(3)
    hosts = [mk(dtype, rng.standard_normal(s)) for s in [(), (3, 4, 5), (1, 1), (2, 0, 3), (17,)]]
    hosts += [mk(dtype, rng.standard_normal(int(n))) for n in rng.integers(0, 40, size=1500)]
    _check(hosts, 1.0)


@pytest.mark.parametrize("scale", [1e30, 1e-30, 1e-42])
def test_magnitudes_whose_squares_leave_f32(scale):
    rng = np.random.default_rng(4)
    for dtype in ("f32", "bf16"):
        h = mk(dtype, rng.uniform(1.0, 2.0, 5000) * scale)
        got, norm = _clip([h], math.inf)
        n = math.sqrt(float(np.sum(vals(h) ** 2)))
        assert abs(norm - n) <= 2.0 ** -19 * n + 2.0 ** -149
        assert np.array_equal(got[0], vals(h))


def test_one_large_among_many_small_and_zeros():
    v = np.full(200000, 1e-4, np.float32)
    v[123456] = 3e4
    _check([mk("f32", v), mk("f32", np.zeros(5000))], 1.0)
    got, norm = _clip([mk("f16", np.zeros(100))], 1.0)
    assert norm == 0.0 and not got[0].any()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_non_finite_gradients_show_in_the_norm(bad):
    for dtype in ("f32", "f16", "bf16"):
        v = np.ones(9000, np.float32)
        v[8500] = bad
        got, norm = _clip([mk(dtype, v), mk("f32", np.ones(3))], 1.0)
        assert math.isnan(norm) if np.isnan(bad) else norm == math.inf
        # max / inf = 0: finite values become 0, inf·0 NaN; a NaN norm makes all NaN
        if np.isnan(bad):
            assert np.isnan(got[0]).all() and np.isnan(got[1]).all()
        else:
            assert np.isnan(got[0][8500]) and not np.delete(got[0], 8500).any() and not got[1].any()
        got, norm = _clip([mk(dtype, v)], math.inf)
        assert np.isnan(got[0]).all() or np.isnan(got[0][8500]) or got[0][8500] == bad


def test_views_and_input_left_alone():
    b = backend()
    rng = np.random.default_rng(5)
    base = mk("f16", rng.standard_normal((40, 300)))
    t = b.fromHost(base)
    flat = b.slice(b.reshape(t, [12000]), [1], [11000])  # dense, 2 bytes past an aligned address
    outs, norm = A.clip_grad_norm(b, [b.transpose(t, [1, 0]), flat], 0.5)
    v = vals(base)
    n = math.sqrt(np.sum(v * v) + np.sum(v.reshape(-1)[1:11000] ** 2))
    f = 0.5 / (n + EPS)
    for o, w in zip(outs, (v.T, v.reshape(-1)[1:11000])):
        g = vals(b.read(o))
        assert g.shape == w.shape and np.all(np.abs(g - w * f) <= (2.0 ** -11 + 2.0 ** -18) * np.abs(w * f) + TINY["f16"])
    assert np.array_equal(b.read(t).data, base.data)


def test_same_bits_and_graph_and_lifetime():
    b = backend()
    rng = np.random.default_rng(6)
    ts = [b.fromHost(mk("bf16", rng.standard_normal(n))) for n in (70000, 12345, 9)]
    f = b.compile(lambda *g: (lambda r: [*r[0], r[1]])(A.clip_grad_norm(b, list(g), 1.0)))
    first = [b.read(v).data for v in f(*ts)]
    for _ in range(3):
        assert all(np.array_equal(p, b.read(q).data) for p, q in zip(first, f(*ts)))
    live = b.stats()
    outs, norm = A.clip_grad_norm(b, ts, 1.0)
    b.dispose(outs[0])
    assert np.array_equal(b.read(outs[1]).data, first[1])  # the allocation lives with the last output
    for t in (outs[1], outs[2], norm):
        b.dispose(t)
    now = b.stats()
    assert now["live_tensors"] == live["live_tensors"] and now["live_bytes"] == live["live_bytes"]


def test_refusals_and_no_gradients():
    b = backend()
    t = b.fromHost(HostTensor("i32", (3,), np.zeros(3, np.int32)))
    with pytest.raises(LayaCudaError, match="f32, f16 or bf16"):
        A.clip_grad_norm(b, [t], 1.0)
    g = b.fromHost(mk("f32", np.ones(4)))
    for bad in (-1.0, math.nan):
        with pytest.raises(LayaCudaError, match="max_norm"):
            A.clip_grad_norm(b, [g], bad)
    outs, norm = A.clip_grad_norm(b, [], 1.0)
    assert outs == [] and float(vals(b.read(norm))) == 0.0
    b.dispose(g)
    with pytest.raises(LayaCudaError, match="dispose"):
        A.clip_grad_norm(b, [g], 1.0)


def test_outputs_as_torch_tensors():
    """The outputs share an allocation: it lives until the last torch tensor
    over it is gone."""
    import torch

    from laya_js_b200 import _lib, interop
    b = backend()
    rng = np.random.default_rng(8)
    hosts = [mk(k, rng.standard_normal(s)) for k, s in (("bf16", (3, 5)), ("f32", (7,)), ("bf16", (0, 4)), ("bf16", (300, 41)), ("f16", ()), ("f32", (2, 2, 2)))]
    want, norm = _want(hosts, 0.5)
    interop.useTorchStream(b)
    try:
        before = b.stats()
        ins = [b.fromHost(h) for h in hosts]
        outs, n = A.clip_grad_norm(b, ins, 0.5)
        ts = [interop.toTorch(b, t) for t in outs[1:]]
        n = interop.toTorch(b, n)
        first = interop.toTorch(b, outs[0])  # after the others
        torch.cuda.synchronize()
        for t, h, w in zip([first, *ts], hosts, want):
            assert tuple(t.shape) == tuple(h.shape) and str(t.dtype) == {"bf16": "torch.bfloat16", "f16": "torch.float16", "f32": "torch.float32"}[h.dtype]
            assert np.all(np.abs(t.double().cpu().numpy() - w) <= (2.0 ** -DIGITS[h.dtype] + 2.0 ** -18) * np.abs(w) + TINY[h.dtype])
        assert abs(float(n) - norm) <= 2.0 ** -19 * norm
        for t in outs:
            b.dispose(t)  # given away: nothing happens
        keep = ts[2]
        copy = keep.clone()
        del ts, first, n, t, outs
        torch.cuda.synchronize()
        assert torch.equal(keep, copy)
        del keep
        for t in ins:
            b.dispose(t)
        after = b.stats()
        assert after["live_tensors"] == before["live_tensors"] and after["live_bytes"] == before["live_bytes"]
    finally:
        torch.cuda.synchronize()
        _lib.call("lc_set_stream", 0)

"""Adapters of many requests beside a shared projection, and their gradients,
against 64 bits: ragged batches with empty requests, rows and adapters that
take no part, odd sizes and every rank range, strided operands, non-finite
rows and adapters that must stay where they are, other streams, recorded
graphs, refusals."""
from __future__ import annotations

import numpy as np
import pytest

from adapters_ref import case, linear_ref, mk, vals
from gpu_util import backend
from laya_js_b200 import adapters as A
from laya_js_b200._lib import LayaCudaError
from laya_js_b200.host import HostTensor

pytestmark = pytest.mark.gpu

# T, K, N, adapters, rank, requests
SHAPES = [
    (0, 64, 64, 2, 4, 3), (1, 64, 64, 1, 1, 1), (3, 768, 2304, 3, 16, 3), (8, 768, 2304, 8, 16, 8), (16, 1152, 768, 5, 64, 16),
    (33, 768, 3, 4, 8, 33), (64, 768, 16, 8, 8, 16), (128, 768, 2304, 4, 16, 1), (129, 64, 72, 2, 17, 2), (255, 200, 200, 3, 12, 9),
    (300, 1001, 777, 7, 12, 23), (500, 768, 768, 64, 8, 200), (513, 1024, 1312, 2, 33, 5), (640, 768, 1536, 3, 100, 4),
    (700, 136, 264, 2, 256, 3), (1000, 72, 5, 3, 5, 40), (2049, 768, 2304, 6, 16, 31), (1537, 2624, 1024, 4, 32, 12), (260, 7, 1, 2, 3, 6),
    (4096, 768, 768, 1, 16, 64), (1290, 768, 1025, 5, 24, 100),
    # long enough that every ring, run and round of tiles goes around more than once
    (70001, 72, 64, 5, 8, 300), (40000, 64, 392, 3, 40, 900), (33333, 328, 72, 40, 16, 3),
]


def _up(b, h):
    return {k: None if t is None else b.fromHost(t) for k, t in h.items()}


def _check(got, want, bound, what):
    backend().flush()  # a pipeline wait that ran out is reported here
    err = np.abs(got - want)
    bad = ~(err <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.max(err / np.maximum(bound, 1e-300)):.3g} bounds at {np.argwhere(bad)[0]}"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,K,N,n,r,requests", SHAPES)
def test_linear_matches_64_bits(dtype, T, K, N, n, r, requests):
    b = backend()
    h, cu, ad = case(dtype, T, K, N, n, r, requests, seed=T + K + N + r, bias=r % 2 == 0)
    t = _up(b, h)
    y = b.read(A.adapter_linear(b, t["x"], t["w"], t["bias"], t["a"], t["bt"], t["scales"], A.AdapterPlan(b, cu, ad, n)))
    assert y.dtype == dtype and y.shape == (T, N)
    want, bound = linear_ref(h, cu, ad, dtype)
    _check(vals(y), want, bound, "y")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,K,N,n,r,requests", SHAPES)
def test_gradients_match_64_bits(dtype, T, K, N, n, r, requests):
    b = backend()
    h, cu, ad = case(dtype, T, K, N, n, r, requests, seed=2 * T + K + N + r)
    t = _up(b, h)
    got = A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], A.AdapterPlan(b, cu, ad, n))
    want, bound = linear_ref(h, cu, ad, dtype, grad=True)
    for name, g, v, m in zip(("dx", "da", "db"), got, want, bound):
        g = b.read(g)
        assert g.dtype == dtype and g.shape == v.shape
        _check(vals(g), v, m, name)
    for k in set(range(n)) - {int(a) for i, a in enumerate(ad) if cu[i + 1] > cu[i]}:
        assert not vals(b.read(got[1]))[k].any() and not vals(b.read(got[2]))[k].any()  # an adapter without rows


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_gradients_against_differences(dtype):
    """loss = Σ y·dy is linear in x, in A and in B: central differences of the
    operator itself in f32 (on values that are exact in the 16-bit type)
    have no truncation error, only the f32 rounding of the two losses."""
    b = backend()
    T, K, N, n, r = 24, 40, 48, 3, 4
    h, cu, ad = case(dtype, T, K, N, n, r, 5, seed=5, bare=0.2)
    h32 = {k: None if v is None else mk("f32", vals(v)) for k, v in h.items()}
    plan = A.AdapterPlan(b, cu, ad, n)
    t = _up(b, h)
    grads = [vals(b.read(g)) for g in A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan)]

    def loss(hh):
        u = _up(b, hh)
        y = vals(b.read(A.adapter_linear(b, u["x"], u["w"], None, u["a"], u["bt"], u["scales"], plan)))
        return float(np.sum(y * vals(hh["dy"])))

    _, bounds = linear_ref(h, cu, ad, dtype, grad=True)
    rng = np.random.default_rng(1)
    step = 0.5
    # each f32 output is off by its own bound; Σ |dy|·bound over the batch, twice, over 2·step
    _, yb = linear_ref(h32, cu, ad, "f32")
    noise = np.sum(np.abs(vals(h["dy"])) * yb) / step
    for name, g, m in zip(("x", "a", "bt"), grads, bounds):
        for _ in range(6):
            i = tuple(rng.integers(0, d) for d in g.shape)
            lo, hi = (vals(h32[name]).copy() for _ in range(2))
            lo[i] -= step
            hi[i] += step
            d = (loss({**h32, name: mk("f32", hi)}) - loss({**h32, name: mk("f32", lo)})) / (2 * step)
            assert abs(d - g[i]) <= m[i] + 2 * noise, (name, i, d, g[i])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_without_a_shared_projection(dtype):
    b = backend()
    h, cu, ad = case(dtype, 300, 768, 264, 3, 16, 7, seed=3, with_w=False)
    t = _up(b, h)
    plan = A.AdapterPlan(b, cu, ad, 3)
    y = vals(b.read(A.adapter_linear(b, t["x"], None, None, t["a"], t["bt"], t["scales"], plan)))
    want, bound = linear_ref(h, cu, ad, dtype)
    _check(y, want, bound, "y")
    got = A.adapter_linear_grad(b, t["dy"], t["x"], None, t["a"], t["bt"], t["scales"], plan)
    want, bound = linear_ref(h, cu, ad, dtype, grad=True)
    for name, g, v, m in zip(("dx", "da", "db"), got, want, bound):
        _check(vals(b.read(g)), v, m, name)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,K,N", [(300, 256, 512), (12, 256, 512), (300, 201, 129), (700, 768, 1280)])
def test_non_finite_values_stay_in_their_request(dtype, T, K, N):
    """Rows of inf and NaN, an adapter of NaN and one of inf: every other
    request's results and every other adapter's gradients keep their bits."""
    b = backend()
    n, r = 4, 8
    h, _, _ = case(dtype, T, K, N, n, r, 1, seed=9)
    edges = [0, T // 7, T // 5, T // 3, T // 2, T // 2 + 1, T]
    cu, ad = np.array(edges, np.int32), np.array([0, 1, 0, 2, 3, 0], np.int32)
    plan = A.AdapterPlan(b, cu, ad, n)
    clean = _up(b, h)
    args = lambda t: (t["w"], None, t["a"], t["bt"], t["scales"], plan)
    y0 = vals(b.read(A.adapter_linear(b, clean["x"], *args(clean))))
    g0 = [vals(b.read(g)) for g in A.adapter_linear_grad(b, clean["dy"], clean["x"], clean["w"], *args(clean)[2:])]
    bad = {k: None if v is None else vals(v).copy() for k, v in h.items()}
    bad["a"][1, :, 3] = np.nan
    bad["bt"][1] = np.inf
    bad["bt"][2, 0, :5] = np.nan
    bad["x"][edges[3]:edges[4]] = np.inf   # the request of adapter 2
    bad["dy"][edges[3]:edges[4]] = np.nan
    t = _up(b, {k: None if v is None else mk("f32" if k == "scales" else dtype, v) for k, v in bad.items()})
    y1 = vals(b.read(A.adapter_linear(b, t["x"], *args(t))))
    g1 = [vals(b.read(g)) for g in A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], *args(t)[2:])]
    ok = np.ones(T, bool)
    ok[edges[1]:edges[2]] = False
    ok[edges[3]:edges[4]] = False
    assert np.array_equal(y0[ok], y1[ok]) and np.array_equal(g0[0][ok], g1[0][ok])
    if edges[2] > edges[1]:
        assert not np.isfinite(y1[edges[1]:edges[2]]).any()
    for k in (0, 3):
        assert np.array_equal(g0[1][k], g1[1][k]) and np.array_equal(g0[2][k], g1[2][k])


def test_only_the_gradients_asked_for():
    b = backend()
    h, cu, ad = case("f16", 200, 64, 96, 2, 8, 3, seed=4)
    t = _up(b, h)
    plan = A.AdapterPlan(b, cu, ad, 2)
    full = [b.read(g).data for g in A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan)]
    for i, k in enumerate(("dx", "da", "db")):
        got = A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan, want=(k,))
        assert [g is not None for g in got] == [j == i for j in range(3)]
        assert np.array_equal(b.read(got[i]).data, full[i])
    assert A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan, want=()) == (None, None, None)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_strided_operands_and_leading_axes(dtype):
    """x and dy as transposed views, w and the up-projections as transposes of
    the other orientation, banks cut out of larger ones: the dense bits."""
    b = backend()
    B, L, K, N, n, r = 3, 50, 72, 96, 3, 8
    h, cu, ad = case(dtype, B * L, K, N, n, r, 4, seed=6, bias=True)
    plan = A.AdapterPlan(b, cu, ad, n)
    t = _up(b, h)
    x3 = b.reshape(t["x"], [B, L, K])
    y0 = b.read(A.adapter_linear(b, x3, t["w"], t["bias"], t["a"], t["bt"], t["scales"], plan))
    assert y0.shape == (B, L, N)
    g0 = [b.read(g) for g in A.adapter_linear_grad(b, b.reshape(t["dy"], [B, L, N]), x3, t["w"], t["a"], t["bt"], t["scales"], plan)]
    assert g0[0].shape == (B, L, K)
    flip = lambda name, perm: b.transpose(b.fromHost(HostTensor(h[name].dtype, tuple(h[name].shape[p] for p in perm), np.ascontiguousarray(h[name].data.transpose(perm)))), np.argsort(perm).tolist())
    xs = b.reshape(flip("x", [1, 0]), [B, L, K])
    w, bt = flip("w", [1, 0]), flip("bt", [0, 2, 1])
    wide = np.concatenate([h["a"].data, h["a"].data], axis=2)
    a = b.slice(b.fromHost(HostTensor(dtype, wide.shape, wide)), [0, 0, K], [n, r, 2 * K])
    dy = b.reshape(flip("dy", [1, 0]), [B, L, N])
    assert np.array_equal(b.read(A.adapter_linear(b, xs, w, t["bias"], a, bt, t["scales"], plan)).data, y0.data)
    for p, q in zip(A.adapter_linear_grad(b, dy, xs, w, a, bt, t["scales"], plan), g0):
        assert np.array_equal(b.read(p).data, q.data)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_operands_off_16_bytes(dtype):
    """Dense operands that start 2 bytes past an aligned address."""
    b = backend()
    T, K, N, n, r = 140, 64, 128, 2, 8
    h, cu, ad = case(dtype, T, K, N, n, r, 3, seed=8)
    plan = A.AdapterPlan(b, cu, ad, n)

    def off(v):
        flat = np.concatenate([v.data.reshape(-1)[:1], v.data.reshape(-1)])
        return b.reshape(b.slice(b.fromHost(HostTensor(dtype, flat.shape, flat)), [1], [flat.size]), list(v.shape))

    t = {k: (None if v is None else b.fromHost(v) if k == "scales" else off(v)) for k, v in h.items()}
    want, bound = linear_ref(h, cu, ad, dtype)
    _check(vals(b.read(A.adapter_linear(b, t["x"], t["w"], None, t["a"], t["bt"], t["scales"], plan))), want, bound, "y")
    want, bound = linear_ref(h, cu, ad, dtype, grad=True)
    for name, g, v, m in zip(("dx", "da", "db"), A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan), want, bound):
        _check(vals(b.read(g)), v, m, name)


@pytest.mark.parametrize("T,K,N,r,requests", [(12, 768, 2304, 16, 12), (700, 768, 768, 16, 9)])
def test_same_bits_every_run_and_in_a_recorded_graph(T, K, N, r, requests):
    b = backend()
    n = 3
    h, cu, ad = case("bf16", T, K, N, n, r, requests, seed=12)
    t = _up(b, h)
    plan = A.AdapterPlan(b, cu, ad, n)

    def both(x, dy):
        y = A.adapter_linear(b, x, t["w"], None, t["a"], t["bt"], t["scales"], plan)
        return [y, *A.adapter_linear_grad(b, dy, x, t["w"], t["a"], t["bt"], t["scales"], plan)]

    first = [b.read(v).data for v in both(t["x"], t["dy"])]
    for _ in range(3):
        assert all(np.array_equal(p, b.read(q).data) for p, q in zip(first, both(t["x"], t["dy"])))
    f = b.compile(both)
    f(t["x"], t["dy"])
    other = mk("bf16", vals(h["x"]) * 0.5)
    f(b.fromHost(other), t["dy"])
    assert all(np.array_equal(p, b.read(q).data) for p, q in zip(first, f(t["x"], t["dy"])))


def test_on_another_stream_and_with_torch_tensors():
    import torch

    from laya_js_b200 import interop
    b = backend()
    h, cu, ad = case("f16", 400, 768, 512, 3, 16, 5, seed=13)
    plan = A.AdapterPlan(b, cu, ad, 3)  # built on the library's own stream
    want, bound = linear_ref(h, cu, ad, "f16")
    tt = {k: torch.from_numpy(v.data).cuda() for k, v in h.items() if v is not None}
    torch.cuda.synchronize()
    try:
        for s in (torch.cuda.default_stream(), torch.cuda.Stream()):
            with torch.cuda.stream(s):
                interop.useTorchStream(b)
                t = {k: interop.fromTorch(b, v + 0) for k, v in tt.items()}  # written on this stream just before
                y = interop.toTorch(b, A.adapter_linear(b, t["x"], t["w"], None, t["a"], t["bt"], t["scales"], plan))
                got = (y + 0).double().cpu().numpy()
            _check(got, want, bound, "y")
        plan.free()
    finally:
        torch.cuda.synchronize()
        from laya_js_b200 import _lib
        _lib.call("lc_set_stream", 0)


def test_nothing_is_left_behind():
    b = backend()
    h, cu, ad = case("bf16", 300, 200, 136, 3, 9, 5, seed=14)
    t = _up(b, h)
    live = b.stats()["live_tensors"]
    for _ in range(3):
        plan = A.AdapterPlan(b, cu, ad, 3)
        y = A.adapter_linear(b, t["x"], t["w"], None, t["a"], t["bt"], t["scales"], plan)
        gs = A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan)
        for v in (y, *gs):
            b.dispose(v)
        plan.free()
    assert b.stats()["live_tensors"] == live


def test_refusals():
    b = backend()
    h, cu, ad = case("f16", 20, 32, 48, 2, 4, 3, seed=15, bias=True)
    t = _up(b, h)
    plan = A.AdapterPlan(b, cu, ad, 2)
    live = b.stats()["live_tensors"]

    def no(match, **kw):
        v = {**t, "plan": plan, **kw}
        with pytest.raises(LayaCudaError, match=match):
            A.adapter_linear(b, v["x"], v["w"], v["bias"], v["a"], v["bt"], v["scales"], v["plan"])

    up = lambda dt, *shape: b.fromHost(mk(dt, np.zeros(shape)))
    made = [up("f32", 48, 32), up("f16", 19, 32), up("f16", 48, 31), up("f16", 3, 4, 32), up("f16", 2, 5, 48), up("f16", 47), up("f32", 3),
            up("f16", 2), up("f16", 2, 257, 32), up("f16", 2, 257, 48), up("f16", 2, 4)]
    no("share a dtype", w=made[0])
    no("19 rows, the plan 20", x=made[1])
    no("expected \\[48,32\\]", w=made[2])
    no("vs b|made for 2", a=made[3])
    no("vs b", bt=made[4])
    no("bias", bias=made[5])
    no("scales", scales=made[6])
    no("scales", scales=made[7])
    no("rank must be", a=made[8], bt=made[9])
    no("a \\[n, r, in\\]", a=made[10])
    ints = b.fromHost(HostTensor("i32", (20, 32), np.zeros((20, 32), np.int32)))
    no("f32, f16 or bf16", x=ints)
    with pytest.raises(LayaCudaError, match="dy"):
        A.adapter_linear_grad(b, t["x"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan)
    with pytest.raises(ValueError, match="unknown"):
        A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan, want=("dw",))
    assert b.stats()["live_tensors"] == live + len(made) + 1
    for cu_, ad_, match in (([1, 20], [0], "start at 0"), ([0, 5, 3], [0, 0], "decrease"), ([0, 5], [2], "adapter 2 of 2"), ([0, 5], [-2], "-2")):
        with pytest.raises(LayaCudaError, match=match):
            A.AdapterPlan(b, cu_, ad_, 2)
    with pytest.raises(ValueError, match="one more"):
        A.AdapterPlan(b, [0, 5], [0, 1], 2)
    dead = A.AdapterPlan(b, cu, ad, 2)
    dead.free()
    no("plan handle", plan=dead)
    with pytest.raises(LayaCudaError, match="out of device memory"):
        from laya_js_b200 import _lib
        _lib.call("lc_debug_set_alloc_cap", 1)
        try:
            A.adapter_linear(b, t["x"], t["w"], None, t["a"], t["bt"], t["scales"], plan)
        finally:
            _lib.call("lc_debug_set_alloc_cap", 0)


def test_inner_values_beyond_f16():
    """u past the largest f16 value (65504) is held in two parts; y is an
    ordinary number."""
    b = backend()
    rng = np.random.default_rng(16)
    for T in (4, 300):
        x = np.abs(rng.standard_normal((T, 64))) + 0.5
        h = {"x": mk("f16", x), "w": None, "bias": None, "a": mk("f16", np.full((1, 2, 64), 1200.0)), "bt": mk("f16", np.full((1, 2, 72), 2.0 ** -12)),
             "scales": mk("f32", np.array([1.0])), "dy": mk("f16", rng.standard_normal((T, 72)))}
        u = vals(h["x"]) @ vals(h["a"])[0].T
        assert u.min() > 65504 and u.max() < 131008
        t = _up(b, h)
        cu, ad = np.array([0, T], np.int32), np.array([0], np.int32)
        y = vals(b.read(A.adapter_linear(b, t["x"], None, None, t["a"], t["bt"], t["scales"], A.AdapterPlan(b, cu, ad, 1))))
        want, bound = linear_ref(h, cu, ad, "f16")
        _check(y, want, bound, "y")


@pytest.mark.parametrize("T,K,N", [(600001, 8, 1), (3, 8, 300001)])
def test_long_and_wide(T, K, N):
    """More groups of rows or columns than one grid axis of 65,535 holds."""
    b = backend()
    h, cu, ad = case("bf16", T, K, N, 2, 2, 3, seed=17)
    t = _up(b, h)
    plan = A.AdapterPlan(b, cu, ad, 2)
    want, bound = linear_ref(h, cu, ad, "bf16")
    _check(vals(b.read(A.adapter_linear(b, t["x"], t["w"], None, t["a"], t["bt"], t["scales"], plan))), want, bound, "y")
    want, bound = linear_ref(h, cu, ad, "bf16", grad=True)
    for name, g, v, m in zip(("dx", "da", "db"), A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan), want, bound):
        _check(vals(b.read(g)), v, m, name)


def test_with_every_kernel_chained():
    """LAYA_CUDA_PDL=1 chains the kernels of consecutive ops too: a stack of
    projections and its gradients keep their bits."""
    import os
    import subprocess
    import sys
    code = """
import sys; sys.path[:0] = ["tests", "."]
import numpy as np
from adapters_ref import case
from laya_js_b200 import createCudaBackend, adapters as A
b = createCudaBackend(0)
out = []
for T, req in ((24, 24), (900, 7)):
    h, cu, ad = case("bf16", T, 256, 256, 3, 16, req, seed=T)
    t = {k: None if v is None else b.fromHost(v) for k, v in h.items()}
    plan = A.AdapterPlan(b, cu, ad, 3)
    x = t["x"]
    for _ in range(6):
        y = A.adapter_linear(b, x, t["w"], None, t["a"], t["bt"], t["scales"], plan)
        gs = A.adapter_linear_grad(b, y, x, t["w"], t["a"], t["bt"], t["scales"], plan)
        c, n = A.clip_grad_norm(b, gs[1:], 1.0)
        x = b.add(b.scale(y, 0.5), gs[0])
    out += [b.read(v).data.astype(np.float64).ravel() for v in (x, y, *c, n)]
b.flush()
sys.stdout.buffer.write(np.concatenate(out).tobytes())
"""
    got = [subprocess.run([sys.executable, "-c", code], env={**os.environ, "LAYA_CUDA_PDL": v}, capture_output=True, check=True, timeout=120).stdout
           for v in ("0", "1")]
    assert len(got[0]) > 0 and got[0] == got[1]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T", [20, 900])
def test_rows_without_an_adapter_over_used_memory(dtype, T):
    """The scratch of rows without an adapter is never written: with NaN left
    in freed memory, nothing of it reaches a result."""
    b = backend()
    h, cu, ad = case(dtype, T, 256, 264, 3, 12, 11, seed=18, bare=0.6)
    t = _up(b, h)
    plan = A.AdapterPlan(b, cu, ad, 3)
    want, bound = linear_ref(h, cu, ad, dtype)
    wg, bg = linear_ref(h, cu, ad, dtype, grad=True)
    for size in (256, 4096, 70000, 1 << 20, 5 << 20):  # what the ops are about to allocate comes from these
        nan = np.full(size // 2, 0x7fff, np.uint16)
        for junk in [b.fromHost(HostTensor("bf16", nan.shape, nan)) for _ in range(3)]:
            b.dispose(junk)
    _check(vals(b.read(A.adapter_linear(b, t["x"], t["w"], None, t["a"], t["bt"], t["scales"], plan))), want, bound, "y")
    for name, g, v, m in zip(("dx", "da", "db"), A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan), wg, bg):
        _check(vals(b.read(g)), v, m, name)


def test_calls_of_every_size_in_turn_and_on_two_streams():
    """Scratch is kept between calls: small and large calls, padded and not,
    alternating on the library's stream and on others, keep their bits."""
    import torch

    from laya_js_b200 import _lib, interop
    b = backend()
    jobs = []
    for T, K, N, r, req in ((4, 64, 72, 8, 4), (900, 201, 129, 12, 7), (3000, 256, 264, 40, 9), (60, 33, 5, 3, 20)):
        h, cu, ad = case("bf16", T, K, N, 3, r, req, seed=T)
        t = _up(b, h)
        jobs.append((t, A.AdapterPlan(b, cu, ad, 3)))

    def run(job):
        t, plan = job
        y = A.adapter_linear(b, t["x"], t["w"], None, t["a"], t["bt"], t["scales"], plan)
        return [y, *A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan)]

    want = [[b.read(v).data for v in run(j)] for j in jobs]
    others = [torch.cuda.Stream(), torch.cuda.default_stream()]
    try:
        for turn in range(6):
            for s in (None, *others):
                torch.cuda.synchronize()
                if s is None:
                    _lib.call("lc_set_stream", 0)
                else:
                    with torch.cuda.stream(s):
                        interop.useTorchStream(b)
                b.flush()
                got = [run(jobs[(i + turn) % len(jobs)]) for i in range(len(jobs))]  # queued one after the other
                for i, vs in enumerate(got):
                    assert all(np.array_equal(b.read(v).data, w) for v, w in zip(vs, want[(i + turn) % len(jobs)]))
    finally:
        torch.cuda.synchronize()
        _lib.call("lc_set_stream", 0)


@pytest.mark.parametrize("T,K,N", [(3000001, 768, 8), (300001, 64, 8192), (3000001, 765, 8)])
def test_more_than_2_31_elements(T, K, N):
    """Operands of 2.3 to 2.5 thousand million values (made and checked on the
    device): the last rows, and an adapter that only they use."""
    import torch

    from laya_js_b200 import _lib, interop
    b = backend()
    r, tail = 4, 700
    g = torch.Generator(device="cuda").manual_seed(T)
    make = lambda *s, std=1.0: (torch.randn(s, generator=g, device="cuda", dtype=torch.bfloat16) * std).to(torch.bfloat16)
    x, dy, w, a, bt = make(T, K), make(T, N), make(N, K, std=0.05), make(2, r, K, std=K ** -0.5), make(2, r, N, std=0.1)
    interop.useTorchStream(b)
    try:
        tx, tdy, tw, ta, tb = (interop.fromTorch(b, v) for v in (x, dy, w, a, bt))
        plan = A.AdapterPlan(b, [0, 1000, T - tail, T], [0, -1, 1], 2)
        y = interop.toTorch(b, A.adapter_linear(b, tx, tw, None, ta, tb, None, plan))
        dx, da, db = (interop.toTorch(b, v) for v in A.adapter_linear_grad(b, tdy, tx, tw, ta, tb, None, plan))
        for rows, k in ((slice(T - tail, T), 1), (slice(0, 1000), 0), (slice(T - tail - 500, T - tail), None)):
            xs, ds, w64 = x[rows].double(), dy[rows].double(), w.double()
            wk = w64 if k is None else w64 + bt[k].double().t() @ a[k].double()
            for got, want in ((y[rows], xs @ wk.t()), (dx[rows], ds @ wk)):
                # bf16: one rounding; f32 sums of at most 8192 terms against the largest result
                assert torch.all((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * want.abs().max() * 0.1)
            if k is not None:
                u, gr = xs @ a[k].double().t(), ds @ bt[k].double().t()
                for got, want in ((da[k], gr.t() @ xs), (db[k], u.t() @ ds)):
                    assert torch.all((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * want.abs().max() * 0.1)
        plan.free()
    finally:
        torch.cuda.synchronize()
        b.flush()
        _lib.call("lc_set_stream", 0)
        del x, dy
        torch.cuda.empty_cache()

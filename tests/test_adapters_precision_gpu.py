"""u and g, the inner values of the adapter operators, keep what f32 holds of
them: whole numbers of up to 20 bits whose differences are the result, training
gradients of small and of scaled losses in f16, inner values far beyond f16."""
from __future__ import annotations

import numpy as np
import pytest

from adapters_ref import mk, vals
from gpu_util import backend
from laya_js_b200 import adapters as A

pytestmark = pytest.mark.gpu

# rows, requests, rank: dot products and tensor cores, every width of the parts (16, 32, 64, 128 and 256 rank rows)
BATCHES = [(12, 12, 8), (24, 3, 24), (700, 9, 8), (700, 60, 24), (900, 5, 40), (600, 200, 40), (640, 4, 100), (300, 2, 256)]


def _batch(rng, T, requests, n, even):
    """Ragged requests; with `even`, of an even number of rows each."""
    cuts = np.sort(rng.integers(0, T // 2 + 1, size=requests - 1)) * 2 if even else np.sort(rng.integers(0, T + 1, size=requests - 1))
    cu = np.concatenate([[0], cuts, [T]]).astype(np.int32)
    ad = rng.integers(-1, n, size=requests).astype(np.int32)
    ad[0] = 0
    return cu, ad


def _pairs(rng, n, r, C, big):
    """A bank of large whole numbers whose rank rows come in pairs that differ in one column, and one of small ones
    whose rank rows come in pairs of opposite sign."""
    large = rng.integers(-big, big + 1, size=(n, r, C[0]))
    small = rng.integers(-1, 2, size=(n, r, C[1])) * (rng.random((n, r, C[1])) < 0.25)
    for j in range(0, r - 1, 2):
        large[:, j + 1] = large[:, j]
        for a in range(n):
            k = rng.integers(0, C[0])
            large[a, j + 1, k] = np.clip(large[a, j, k] + rng.choice([-1, 1]), -big, big)
        small[:, j + 1] = -small[:, j]
    if r % 2:
        large[:, -1] = rng.integers(-1, 2, size=(n, C[0]))
    return large, small


def _rounded(dtype, v):
    return vals(mk(dtype, v))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,requests,r", BATCHES)
@pytest.mark.parametrize("with_w", [False, True])
def test_forward_keeps_every_bit_of_u(dtype, T, requests, r, with_w):
    """u has 17 to 20 bits and y is a difference of them: every sum is a whole
    number below 2^24, which f32 holds in any order, so y is the exact result
    rounded once. (16 bits of u are off by whole numbers; past 131,008, which
    a third of u is, two f16 parts have no value.)"""
    b = backend()
    rng = np.random.default_rng(T + r)
    K, N, n = 768, 200, 3
    cu, ad = _batch(rng, T, requests, n, False)
    a, bt = _pairs(rng, n, r, (K, N), 255)
    x = rng.integers(-63, 64, size=(T, K))
    w = rng.integers(-1, 2, size=(N, K)) * (rng.random((N, K)) < 0.1)
    want, most, largest = (x @ w.T if with_w else np.zeros((T, N), np.int64)), np.zeros((T, N), np.int64), 0
    for i, k in enumerate(ad):
        if k >= 0:
            s = slice(cu[i], cu[i + 1])
            u = x[s] @ a[k].T
            want[s] += u @ bt[k]
            most[s] = np.abs(u) @ np.abs(bt[k])
            largest = max(largest, np.abs(u).max(initial=0))
    assert most.max() + 63 * K < 2 ** 24 and np.abs(x).max() * np.abs(a).max() * K < 2 ** 24 and largest > 131008
    t = {k: b.fromHost(mk(dtype, v)) for k, v in (("x", x), ("w", w), ("a", a), ("bt", bt))}
    y = A.adapter_linear(b, t["x"], t["w"] if with_w else None, None, t["a"], t["bt"], None, A.AdapterPlan(b, cu, ad, n))
    assert np.array_equal(vals(b.read(y)), _rounded(dtype, want))


@pytest.mark.parametrize("T,requests,r", BATCHES)
@pytest.mark.parametrize("dtype,unit_dy,unit_b,unit_x", [("bf16", 1, 1, 1), ("f16", 1, 1, 1), ("f16", 2.0 ** -20, 2.0 ** -8, 2.0 ** 8),
                                                         ("f16", 2.0 ** 8, 2.0 ** 6, 2.0 ** -12)])
def test_gradients_keep_every_bit_of_g(dtype, T, requests, r, unit_dy, unit_b, unit_x):
    """dx and dA are differences of large g (dx over pairs of rank rows, dA
    over pairs of batch rows whose x have opposite signs), in units from 2^-28
    (a g of 1e-3 to 1e-9) to 2^14 (a g of 1e10): exact results rounded once."""
    b = backend()
    rng = np.random.default_rng(T + r + 1)
    K, N, n = 200, 768, 3
    cu, ad = _batch(rng, T, requests, n, True)
    bt, a = _pairs(rng, n, r, (N, K), 255)
    dy = rng.integers(-63, 64, size=(T, N))
    x = rng.integers(-1, 2, size=(T, K)) * (rng.random((T, K)) < 0.1)
    for i in range(0, T, 2):
        dy[i + 1] = dy[i]
        k = rng.integers(0, N, size=3)
        dy[i + 1, k] = np.clip(dy[i, k] + rng.choice([-1, 1], size=3), -63, 63)
        x[i + 1] = -x[i]
    dx, da = np.zeros((T, K), np.int64), np.zeros((n, r, K), np.int64)
    most, most_a = np.zeros((T, K), np.int64), np.zeros((n, r, K), np.int64)
    for i, k in enumerate(ad):
        if k >= 0:
            s = slice(cu[i], cu[i + 1])
            g = dy[s] @ bt[k].T
            dx[s] = g @ a[k]
            da[k] += g.T @ x[s]
            most[s] = np.abs(g) @ np.abs(a[k])
            most_a[k] += np.abs(g).T @ np.abs(x[s])
    assert max(most.max(), most_a.max(), 63 * 255 * N) < 2 ** 24
    t = {k: b.fromHost(mk(dtype, v)) for k, v in (("dy", dy * unit_dy), ("x", x * unit_x), ("a", a * unit_x), ("bt", bt * unit_b))}
    for v, e in ((t["dy"], dy * unit_dy), (t["x"], x * unit_x), (t["bt"], bt * unit_b)):
        assert np.array_equal(vals(b.read(v)), e)
    got = A.adapter_linear_grad(b, t["dy"], t["x"], None, t["a"], t["bt"], None, A.AdapterPlan(b, cu, ad, n), want=("dx", "da"))
    unit = unit_dy * unit_b * unit_x
    for g, want in ((got[0], dx), (got[1], da)):
        assert np.array_equal(vals(b.read(g)), _rounded(dtype, want * unit))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,requests,r", BATCHES)
def test_gradients_keep_every_bit_of_u(dtype, T, requests, r):
    """dB is a difference of large u over pairs of rows with dy of opposite sign."""
    b = backend()
    rng = np.random.default_rng(T + r + 2)
    K, N, n = 768, 200, 3
    cu, ad = _batch(rng, T, requests, n, True)
    a, bt = _pairs(rng, n, r, (K, N), 255)
    x = rng.integers(-63, 64, size=(T, K))
    dy = rng.integers(-1, 2, size=(T, N)) * (rng.random((T, N)) < 0.1)
    for i in range(0, T, 2):
        x[i + 1] = x[i]
        k = rng.integers(0, K, size=3)
        x[i + 1, k] = np.clip(x[i, k] + rng.choice([-1, 1], size=3), -63, 63)
        dy[i + 1] = -dy[i]
    db, most = np.zeros((n, r, N), np.int64), np.zeros((n, r, N), np.int64)
    for i, k in enumerate(ad):
        if k >= 0:
            s = slice(cu[i], cu[i + 1])
            u = x[s] @ a[k].T
            db[k] += u.T @ dy[s]
            most[k] += np.abs(u).T @ np.abs(dy[s])
    assert max(most.max(), 63 * 255 * K) < 2 ** 24
    t = {k: b.fromHost(mk(dtype, v)) for k, v in (("dy", dy), ("x", x), ("a", a), ("bt", bt))}
    got = A.adapter_linear_grad(b, t["dy"], t["x"], None, t["a"], t["bt"], None, A.AdapterPlan(b, cu, ad, n), want=("db",))
    assert np.array_equal(vals(b.read(got[2])), _rounded(dtype, db))


@pytest.mark.parametrize("dy,up", [(1e-4, 0.02), (1e-5, 0.02), (3e-6, 0.02), (1e-3, 1e-4), (1e-4, 1e-3), (1e-6, 1e-2)])
def test_f16_gradients_of_small_losses(dy, up):
    """dA and dB of 4096 rows against 64 bits: as far off as the one rounding
    to f16 (whose subnormals these reach) and f32 sums, whose error is below
    2^-17 of the norm (a g is off by at most sqrt(768)·2^-24 of the norm of
    its products, random over the rows)."""
    b = backend()
    rng = np.random.default_rng(7)
    T, K, N, r = 4096, 768, 768, 8
    h = {"x": mk("f16", rng.standard_normal((T, K))), "dy": mk("f16", rng.standard_normal((T, N)) * dy),
         "a": mk("f16", rng.standard_normal((1, r, K)) * K ** -0.5), "bt": mk("f16", rng.standard_normal((1, r, N)) * up)}
    v = {k: vals(t) for k, t in h.items()}
    t = {k: b.fromHost(s) for k, s in h.items()}
    _, da, db = A.adapter_linear_grad(b, t["dy"], t["x"], None, t["a"], t["bt"], None, A.AdapterPlan(b, [0, T], [0], 1), want=("da", "db"))
    g, u = v["dy"] @ v["bt"][0].T, v["x"] @ v["a"][0].T
    for got, want in ((da, g.T @ v["x"]), (db, u.T @ v["dy"])):
        once = np.linalg.norm(_rounded("f16", want) - want)
        assert np.linalg.norm(vals(b.read(got))[0] - want) <= 1.05 * once + 2.0 ** -17 * np.linalg.norm(want)


@pytest.mark.parametrize("T", [4, 300])
def test_f16_inner_values_of_any_size(T):
    """u of 1e5 to 6e10 beside adapters of 2^-24 to 2^-8: y is an ordinary number. g of 1e10 with x of 2^-20: dA is one."""
    b = backend()
    rng = np.random.default_rng(8)
    cu, ad = [0, T // 2, T], [0, 1]
    plan = A.AdapterPlan(b, cu, ad, 2)
    x, a = rng.uniform(0.5, 1, (T, 64)), rng.uniform(0.5, 1, (2, 2, 64))
    x[T // 2:] *= 3e4
    x[:T // 2] *= 60
    a[0] *= 60
    a[1] *= 6e4
    bt = np.stack([np.full((2, 72), 2.0 ** -8), np.full((2, 72), 2.0 ** -22)])
    h = {k: mk("f16", v) for k, v in (("x", x), ("a", a), ("bt", bt))}
    v, t = {k: vals(s) for k, s in h.items()}, {k: b.fromHost(s) for k, s in h.items()}
    y = vals(b.read(A.adapter_linear(b, t["x"], None, None, t["a"], t["bt"], None, plan)))
    for i in (0, 1):
        s = slice(cu[i], cu[i + 1])
        u = v["x"][s] @ v["a"][i].T
        assert u.max() > (1e5 if i == 0 else 2e10)
        want = u @ v["bt"][i]
        assert want.max() < 65504
        # one rounding to f16; f32 sums of positive terms
        assert np.all(np.abs(y[s] - want) <= (2.0 ** -11 + 2.0 ** -16) * want)
    # the same numbers as dy and B give g; x of 2^-20
    small = mk("f16", np.full((T, 72), 2.0 ** -20))
    da = A.adapter_linear_grad(b, t["x"], b.fromHost(small), None, t["bt"], t["a"], None, plan, want=("da",))[1]
    da = vals(b.read(da))
    for i in (0, 1):
        s = slice(cu[i], cu[i + 1])
        g = v["x"][s] @ v["a"][i].T
        want = g.T @ vals(small)[s]
        if want.max() < 65504 and g.max() < 3.4e10:
            assert np.all(np.abs(da[i] - want) <= (2.0 ** -11 + 2.0 ** -16) * want + 2.0 ** -25)


def test_f16_gradients_are_the_exact_ones_rounded_but_for_few():
    """The f32 sums end a little below the exact value (the tensor cores cut
    where they add): g by half a unit of 2^-24 of the running half in each of
    48 steps, dA in each of 16 more, 2^-20 together. A value moved by that
    rounds to the other f16 neighbour in 2^-20 / (1.4 * 2^-11) = 0.14 % of the
    cases; twice that is allowed. Errors of 2^-18 would show as 0.6 %."""
    b = backend()
    rng = np.random.default_rng(9)
    T, K, N, n, r = 1000, 768, 768, 4, 32
    cu, ad = [0, 250, 500, 750, T], [0, 1, 2, 3]
    h = {"x": mk("f16", rng.standard_normal((T, K))), "dy": mk("f16", rng.standard_normal((T, N)) * 0.05),
         "a": mk("f16", rng.standard_normal((n, r, K)) * K ** -0.5), "bt": mk("f16", rng.standard_normal((n, r, N)) * 0.02)}
    v, t = {k: vals(s) for k, s in h.items()}, {k: b.fromHost(s) for k, s in h.items()}
    _, da, db = A.adapter_linear_grad(b, t["dy"], t["x"], None, t["a"], t["bt"], None, A.AdapterPlan(b, cu, ad, n), want=("da", "db"))
    for got, pick in ((da, lambda s, k: (v["dy"][s] @ v["bt"][k].T).T @ v["x"][s]), (db, lambda s, k: (v["x"][s] @ v["a"][k].T).T @ v["dy"][s])):
        want = np.stack([pick(slice(cu[k], cu[k + 1]), k) for k in range(n)])
        assert np.mean(vals(b.read(got)) != _rounded("f16", want)) <= 2 * 2.0 ** -20 / (1.4 * 2.0 ** -11)

"""The adapter operators in 64 bits (numpy), request by request, and the error
bounds their GPU forms are held to."""
from __future__ import annotations

import numpy as np

from laya_js_b200.host import HostTensor, f32_to_bf16_bits, to_f32

DIGITS = {"f32": 24, "f16": 11, "bf16": 8}  # significand bits: rounding to nearest is off by 2^-DIGITS at most
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}  # half the smallest subnormal


def mk(dtype, a):
    a = np.ascontiguousarray(a, np.float32)
    if dtype == "f16":
        return HostTensor("f16", a.shape, a.astype(np.float16))
    if dtype == "bf16":
        return HostTensor("bf16", a.shape, f32_to_bf16_bits(a))
    return HostTensor("f32", a.shape, a)


def vals(h):
    return to_f32(h).astype(np.float64)


def case(dtype, T, K, N, n, r, requests, seed, with_w=True, bias=False, bare=0.25):
    """Inputs of a ragged batch (values as stored, in 64 bits) with empty requests and bare rows."""
    rng = np.random.default_rng(seed)
    cuts = np.sort(rng.integers(0, T + 1, size=requests - 1)) if requests else np.zeros(0, int)
    cu = np.concatenate([[0], cuts, [T]]).astype(np.int32) if requests else np.zeros(1, np.int32)
    ad = rng.integers(0, n, size=requests).astype(np.int32) if n else np.full(requests, -1, np.int32)
    ad[rng.random(requests) < bare] = -1
    h = {"x": mk(dtype, rng.standard_normal((T, K))), "w": mk(dtype, rng.standard_normal((N, K)) * 0.05) if with_w else None,
         "bias": mk(dtype, rng.standard_normal(N)) if bias else None, "a": mk(dtype, rng.standard_normal((n, r, K)) * K ** -0.5),
         "bt": mk(dtype, rng.standard_normal((n, r, N)) * 0.1), "scales": mk("f32", rng.uniform(0.5, 2.0, n)),
         "dy": mk(dtype, rng.standard_normal((T, N)))}
    return h, cu, ad


def _rows(cu, ad):
    for i, a in enumerate(ad):
        if a >= 0 and cu[i + 1] > cu[i]:
            yield slice(int(cu[i]), int(cu[i + 1])), int(a)


def linear_ref(h, cu, ad, dtype, grad=False):
    """(values, bounds): each value's bound is the rounding of the result to its
    dtype, the f32 sums (worst case: their length times 2^-23 of the sum of
    magnitudes) and, for 16-bit dtypes, u and g held in at least 16 bits."""
    v = {k: None if t is None else vals(t) for k, t in h.items()}
    x, w, a, bt, s, dy = v["x"], v["w"], v["a"], v["bt"], v["scales"], v["dy"]
    T, K = x.shape
    N, r = bt.shape[2], bt.shape[1]
    keep = 0.0 if dtype == "f32" else 2.0 ** -16
    out = 2.0 ** -DIGITS[dtype]

    def bound(val, mag, n):
        return out * np.abs(val) + (n * 2.0 ** -23 + keep) * mag * (1 + out) + TINY[dtype] * (1 + n)

    if not grad:
        y = x @ w.T if w is not None else np.zeros((T, N))
        m = np.abs(x) @ np.abs(w).T if w is not None else np.zeros((T, N))
        if v["bias"] is not None:
            y, m = y + v["bias"], m + np.abs(v["bias"])
        for rows, k in _rows(cu, ad):
            y[rows] += s[k] * (x[rows] @ a[k].T) @ bt[k]
            m[rows] += s[k] * (np.abs(x[rows]) @ np.abs(a[k]).T) @ np.abs(bt[k])
        return y, bound(y, m, 2 * K + r)
    dx = dy @ w if w is not None else np.zeros((T, K))
    mx = np.abs(dy) @ np.abs(w) if w is not None else np.zeros((T, K))
    da, db, ma, mb = np.zeros_like(a), np.zeros_like(bt), np.zeros_like(a), np.zeros_like(bt)
    for rows, k in _rows(cu, ad):
        g, gm = s[k] * dy[rows] @ bt[k].T, s[k] * np.abs(dy[rows]) @ np.abs(bt[k]).T
        u, um = s[k] * x[rows] @ a[k].T, s[k] * np.abs(x[rows]) @ np.abs(a[k]).T
        dx[rows] += g @ a[k]
        mx[rows] += gm @ np.abs(a[k])
        da[k] += g.T @ x[rows]
        ma[k] += gm.T @ np.abs(x[rows])
        db[k] += u.T @ dy[rows]
        mb[k] += um.T @ np.abs(dy[rows])
    return (dx, da, db), (bound(dx, mx, 2 * N + r), bound(da, ma, N + T), bound(db, mb, K + T))

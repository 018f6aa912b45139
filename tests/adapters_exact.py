"""Whole-number cases of the adapter operators: every sum is a whole number
below 2^24 in any order, so f32 holds it exactly and each result is the exact
one rounded once to its dtype."""
from __future__ import annotations

import numpy as np

from adapters_ref import mk, vals


def _sparse(rng, shape, most, density):
    v = rng.integers(1, most + 1, size=shape) * rng.choice([-1, 1], size=shape)
    return (v * (rng.random(shape) < density)).astype(np.float64)


def whole_case(T, K, N, n, r, requests, seed, bare=0.25):
    """(inputs as float64 whole numbers, cu_rows, adapters); the widths' densities keep sums of thousands of terms small."""
    rng = np.random.default_rng(seed)
    cuts = np.sort(rng.integers(0, T + 1, size=requests - 1))
    cu = np.concatenate([[0], cuts, [T]]).astype(np.int32)
    ad = rng.integers(0, n, size=requests).astype(np.int32)
    ad[rng.random(requests) < bare] = -1
    in_k, in_n = min(1.0, 64 / K), min(1.0, 64 / N)
    v = {"x": _sparse(rng, (T, K), 2, 0.5), "w": _sparse(rng, (N, K), 2, in_k), "a": _sparse(rng, (n, r, K), 2, in_k),
         "bt": _sparse(rng, (n, r, N), 2, in_n), "dy": _sparse(rng, (T, N), 2, 0.5), "bias": _sparse(rng, (N,), 9, 1.0),
         "scales": 2.0 ** rng.integers(0, 3, size=n)}
    return v, cu, ad


def rows_of(cu, ad):
    for i, a in enumerate(ad):
        if a >= 0 and cu[i + 1] > cu[i]:
            yield slice(int(cu[i]), int(cu[i + 1])), int(a)


def exact(v, cu, ad, skip=None):
    """({y, dx, da, db}, the largest sum of magnitudes anywhere); ``skip``: rows whose part in da and db is left out."""
    f = {k: t.astype(np.float64) for k, t in v.items()}
    mag = {k: np.abs(t) for k, t in f.items()}
    out, most = {}, []
    for q, m in ((f, None), (mag, most)):
        y, dx = q["x"] @ q["w"].T + q["bias"], q["dy"] @ q["w"]
        da, db = np.zeros_like(q["a"]), np.zeros_like(q["bt"])
        for rows, k in rows_of(cu, ad):
            # (magnitudes of what is summed: u and g themselves are single values by then)
            u = f["scales"][k] * f["x"][rows] @ f["a"][k].T
            g = f["scales"][k] * f["dy"][rows] @ f["bt"][k].T
            if m is not None:
                m.append((f["scales"][k] * q["x"][rows] @ q["a"][k].T).max())
                m.append((f["scales"][k] * q["dy"][rows] @ q["bt"][k].T).max())
                u, g = np.abs(u), np.abs(g)
            y[rows] += u @ q["bt"][k]
            dx[rows] += g @ q["a"][k]
            if skip is not None:
                u, g = u.copy(), g.copy()
                lo, hi = (min(max(e - rows.start, 0), u.shape[0]) for e in skip)
                u[lo:hi] = g[lo:hi] = 0
            da[k] += g.T @ q["x"][rows]
            db[k] += u.T @ q["dy"][rows]
        if m is None:
            out = {"y": y, "dx": dx, "da": da, "db": db}
        else:
            m += [t.max(initial=0) for t in (y, dx, da, db)]
    return out, max(most)


def rounded(dtype, v):
    return vals(mk(dtype, v))

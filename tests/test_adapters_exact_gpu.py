"""The adapter operators on whole numbers, bit for bit: a block of rows that is
left out or counted twice, a partial that is lost or a stage that is stale
changes whole numbers, however long the sum is. The CPU test shows that the
comparison sees one block of 64 rows at every shape."""
from __future__ import annotations

import numpy as np
import pytest

from adapters_exact import exact, rounded, rows_of, whole_case
from adapters_ref import mk, vals
from gpu_util import backend
from laya_js_b200 import adapters as A
from test_adapters_gpu import SHAPES

LONG = [s for s in SHAPES if s[0]]


@pytest.mark.parametrize("T,K,N,n,r,requests", LONG)
def test_the_comparison_sees_one_block_of_rows(T, K, N, n, r, requests):
    v, cu, ad = whole_case(T, K, N, n, r, requests, seed=T + K + r)
    full, most = exact(v, cu, ad)
    assert most < 2 ** 24
    blocks = [(t, min(t + 64, rows.stop)) for rows, _ in rows_of(cu, ad) for t in range(rows.start, rows.stop, 64)]
    for skip in (blocks[0], blocks[len(blocks) // 2], blocks[-1]) if blocks else ():
        less, _ = exact(v, cu, ad, skip=skip)
        for k in ("da", "db"):
            if skip[1] - skip[0] < 8 and np.array_equal(less[k], full[k]):
                continue  # (a few rows of zeros)
            for dtype in ("f16", "bf16", "f32"):
                # far more than one value: of what 64 rows add, more than a tenth shows in bf16's 8 bits
                assert np.count_nonzero(rounded(dtype, less[k]) != rounded(dtype, full[k])) >= min(10, np.count_nonzero(less[k] != full[k]) // 10)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,K,N,n,r,requests", LONG)
def test_whole_numbers_bit_for_bit(dtype, T, K, N, n, r, requests):
    b = backend()
    v, cu, ad = whole_case(T, K, N, n, r, requests, seed=T + K + r)
    want, most = exact(v, cu, ad)
    assert most < 2 ** 24
    t = {k: b.fromHost(mk("f32" if k == "scales" else dtype, a)) for k, a in v.items()}
    plan = A.AdapterPlan(b, cu, ad, n)
    got = {"y": A.adapter_linear(b, t["x"], t["w"], t["bias"], t["a"], t["bt"], t["scales"], plan)}
    got.update(zip(("dx", "da", "db"), A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan)))
    for k, w in want.items():
        g, w = vals(b.read(got[k])), rounded(dtype, w)
        assert np.array_equal(g, w), f"{k}: {np.count_nonzero(g != w)} of {w.size} differ, first at {np.argwhere(g != w)[0]}"
    b.flush()
    for x in (*t.values(), *got.values()):
        b.dispose(x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,K,N,r", [(20, 256, 264, 8), (900, 256, 264, 8), (900, 256, 264, 40), (900, 201, 129, 20)])
def test_nan_left_in_the_kept_scratch_reaches_nothing(dtype, T, K, N, r):
    """The scratch of a call is kept for the next one. A call whose u and g are
    NaN in every row fills it; rows without an adapter, which the next call
    does not write, start from that."""
    b = backend()
    v, cu, ad = whole_case(T, K, N, 3, r, 11, seed=T + r, bare=0.6)
    want, _ = exact(v, cu, ad)
    t = {k: b.fromHost(mk("f32" if k == "scales" else dtype, a)) for k, a in v.items()}
    nan = {k: b.fromHost(mk(dtype, np.full(v[k].shape, np.nan))) for k in ("x", "dy", "a", "bt", "w")}
    full, plan = A.AdapterPlan(b, [0, T], [1], 3), A.AdapterPlan(b, cu, ad, 3)

    def both(s, plan):
        y = A.adapter_linear(b, s["x"], s["w"], None if s is nan else t["bias"], s["a"], s["bt"], t["scales"], plan)
        return dict(zip(("y", "dx", "da", "db"), (y, *A.adapter_linear_grad(b, s["dy"], s["x"], s["w"], s["a"], s["bt"], t["scales"], plan))))
    for _ in range(3):  # (it grows to what the calls before have asked for)
        for x in both(nan, full).values():
            assert np.isnan(vals(b.read(x))).any()
            b.dispose(x)
    # each operator right after its NaN form: the scratch is laid out alike
    for names, call in ((("y",), lambda s, p: (A.adapter_linear(b, s["x"], s["w"], None if s is nan else t["bias"], s["a"], s["bt"], t["scales"], p),)),
                        (("dx", "da", "db"), lambda s, p: A.adapter_linear_grad(b, s["dy"], s["x"], s["w"], s["a"], s["bt"], t["scales"], p))):
        for x in call(nan, full):
            b.dispose(x)
        for k, x in zip(names, call(t, plan)):
            assert np.array_equal(vals(b.read(x)), rounded(dtype, want[k])), k
            b.dispose(x)

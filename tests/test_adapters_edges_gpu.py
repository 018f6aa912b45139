"""Banks of no adapters, and batches in which no row has one: the shared
projection alone, and gradients of zeros."""
from __future__ import annotations

import numpy as np
import pytest

from adapters_exact import exact, rounded, whole_case
from adapters_ref import mk, vals
from gpu_util import backend
from laya_js_b200 import _lib, interop
from laya_js_b200 import adapters as A
from laya_js_b200.host import HostTensor

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,K,N", [(20, 64, 72), (300, 768, 768), (1500, 768, 1280), (300, 201, 129)])
@pytest.mark.parametrize("n,through_torch", [(0, False), (0, True), (3, False)])
def test_no_row_has_an_adapter(dtype, T, K, N, n, through_torch):
    import torch
    b = backend()
    v, _, _ = whole_case(T, K, N, 3, 8, 5, seed=T)
    cu, ad = [0, 5, T], [-1, -1]
    want, _ = exact(v, np.array(cu), np.array(ad))
    v = {k: (a[:n] if k in ("a", "bt", "scales") else a) for k, a in v.items()}
    t = {k: b.fromHost(mk("f32" if k == "scales" else dtype, a)) for k, a in v.items()}
    try:
        if through_torch:  # whose tensors without elements have no address
            interop.useTorchStream(b)
            kind = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
            t = {k: interop.fromTorch(b, torch.from_numpy(a).cuda().to(kind["f32" if k == "scales" else dtype])) for k, a in v.items()}
        plan = A.AdapterPlan(b, cu, ad, n)
        got = {"y": A.adapter_linear(b, t["x"], t["w"], t["bias"], t["a"], t["bt"], t["scales"], plan)}
        got.update(zip(("dx", "da", "db"), A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan)))
        for k, x in got.items():
            g = vals(b.read(x))
            if k in ("da", "db"):
                assert g.shape == v["a" if k == "da" else "bt"].shape and not g.any()
            else:
                assert np.array_equal(g, rounded(dtype, want[k])), k
        b.flush()
    finally:
        torch.cuda.synchronize()
        _lib.call("lc_set_stream", 0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_no_rows_at_all(dtype):
    b = backend()
    t = {"x": mk(dtype, np.zeros((0, 64))), "w": mk(dtype, np.ones((72, 64))), "a": mk(dtype, np.ones((2, 4, 64))), "bt": mk(dtype, np.ones((2, 4, 72))),
         "dy": mk(dtype, np.zeros((0, 72)))}
    t = {k: b.fromHost(h) for k, h in t.items()}
    for cu, ad in (([0], []), ([0, 0, 0], [1, -1])):
        plan = A.AdapterPlan(b, cu, ad, 2)
        assert A.adapter_linear(b, t["x"], t["w"], None, t["a"], t["bt"], None, plan).shape == (0, 72)
        dx, da, db = A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], None, plan)
        assert dx.shape == (0, 64) and not vals(b.read(da)).any() and not vals(b.read(db)).any()
    clipped, norm = A.clip_grad_norm(b, [b.fromHost(HostTensor("f32", (0, 3), np.zeros((0, 3), np.float32)))], 1.0)
    assert clipped[0].shape == (0, 3) and float(vals(b.read(norm))) == 0.0

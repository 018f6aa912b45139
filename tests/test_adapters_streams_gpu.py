"""Adapter calls from two threads, one after the other, each on its own
per-thread default stream: one handle value, two streams."""
from __future__ import annotations

import threading

import numpy as np
import pytest

from adapters_ref import case
from gpu_util import backend
from laya_js_b200 import _lib
from laya_js_b200 import adapters as A

pytestmark = pytest.mark.gpu

PER_THREAD = 2  # cudaStreamPerThread


@pytest.mark.parametrize("T", [12, 900])
def test_two_threads_on_their_default_streams(T):
    b = backend()
    jobs = []
    for seed in (1, 2):
        h, cu, ad = case("bf16", T, 256, 264, 3, 8, 7, seed=seed)
        jobs.append(({k: None if v is None else b.fromHost(v) for k, v in h.items()}, cu, ad))
    # (whatever the first thread queued may still run when the second one calls)
    def run(job, plan):
        t = job[0]
        return [A.adapter_linear(b, t["x"], t["w"], None, t["a"], t["bt"], t["scales"], plan),
                *A.adapter_linear_grad(b, t["dy"], t["x"], t["w"], t["a"], t["bt"], t["scales"], plan)]
    plans = [A.AdapterPlan(b, job[1], job[2], 3) for job in jobs]
    want = [[b.read(v).data for v in run(job, plan)] for job, plan in zip(jobs, plans)]
    b.flush()
    got, own = [], []

    def work(i):
        _lib.call("lc_set_stream", PER_THREAD)
        if i == 0:
            own.append(A.AdapterPlan(b, jobs[1][1], jobs[1][2], 3))  # built here, first used by the other thread
        for _ in range(20):
            out = run(jobs[i], plans[i] if i == 0 else own[0])
        got.append(out)
    try:
        for i in (0, 1):
            t = threading.Thread(target=work, args=(i,))
            t.start()
            t.join()
        import torch
        torch.cuda.synchronize()
        _lib.call("lc_set_stream", 0)
        for vs, ws in zip(got, want):
            assert all(np.array_equal(b.read(v).data, w) for v, w in zip(vs, ws))
    finally:
        _lib.call("lc_set_stream", 0)
        b.flush()

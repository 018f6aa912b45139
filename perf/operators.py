"""Cases that measure the adapter operators and gradient clipping.

Three operators, as a program that serves and trains low-rank adapters of many
tenants beside one shared encoder uses them:

- ``linear``  y[t] = W·x[t] (+ bias) + s_a · Bᵀ_a·(A_a·x[t]), a = the adapter of row t (none: the shared
              projection alone); x [T, K], W [N, K], A [n, r, K], B [n, r, N], s [n];
- ``grad``    its gradients dx [T, K], dA [n, r, K], dB [n, r, N] for dy [T, N] (W, bias and s are frozen);
- ``clip``    the global norm over many gradient tensors, and the tensors scaled to at most ``max_norm``.

``run`` computes them in elementary torch operations in 32 bits, or with the
framework's own operators where ``own`` is true. ``exact`` is the definition
in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# The draws stay within the work of the largest listed cases (rows·K·N products, gradient elements).
_MOST_MKN = 40000 * 1024 * 5248
_MOST_ELEMENTS = 44 * 32 * 16 * 2304
_EPS = 1e-6  # added to the norm before dividing, as gradient clipping usually does


def listed():
    def rows(name, op, dtype, T, requests, adapters, rank, K, N, bare=0.0, bias=False):
        return {"name": name, "op": op, "dtype": dtype, "rows": T, "requests": requests, "adapters": adapters, "rank": rank,
                "K": K, "N": N, "bare": bare, "bias": bias}

    return [
        # one row per request (the [CLS] rows, or one new token each), a small batch: latency
        rows("linear-8-rows", "linear", "bf16", 8, 8, 8, 16, 768, 2304),
        # the [CLS] rows of a full batch through a small classifier head, an adapter per tenant
        rows("linear-head-256-rows", "linear", "f16", 256, 256, 64, 8, 768, 16, bare=0.125, bias=True),
        # one 128-token prompt through the fused q/k/v projection: latency of a single request
        rows("linear-1-prompt", "linear", "f16", 128, 1, 4, 16, 768, 2304),
        # a ragged batch with sizes that fit no tile, and a rank that fits no vector
        rows("linear-odd", "linear", "bf16", 1537, 23, 7, 12, 1001, 777, bare=0.25, bias=True),
        # the batch of 256 prompts of 32 to 512 tokens through the q/k/v projection
        rows("linear-256-prompts", "linear", "f16", 69135, 256, 32, 16, 768, 2304, bare=0.125),
        # the large shape: prompts of hundreds of tokens through the gated MLP's input projection
        rows("linear-large", "linear", "bf16", 40000, 64, 16, 32, 1024, 5248),
        # training a head: 64 pooled rows, few classes
        rows("grad-head-64-rows", "grad", "bf16", 64, 16, 8, 8, 768, 16),
        # one micro-batch of a few prompts through the attention output projection
        rows("grad-4-prompts", "grad", "f16", 997, 4, 4, 8, 768, 768),
        # a training batch through the MLP's output projection, one adapter for most of it
        rows("grad-64-prompts", "grad", "bf16", 16384, 64, 3, 16, 1152, 768, bare=0.125),
        # the large shape
        rows("grad-large", "grad", "bf16", 40000, 64, 16, 32, 1024, 5248),
        # the adapters of one head, in 32 bits: latency
        {"name": "clip-head", "op": "clip", "dtype": "f32", "tensors": 4, "adapters": 8, "rank": 8, "K": 768, "N": 768, "norm": 1.0},
        # A and B of the q/k/v projection in each of 22 layers, 32 tenants
        {"name": "clip-22-layers", "op": "clip", "dtype": "bf16", "tensors": 44, "adapters": 32, "rank": 16, "K": 768, "N": 2304, "norm": 1.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: mostly multiples of 64 or 8, one in four whatever comes."""
    v = _log_int(rng, lo, hi)
    q = min(rng.choice((64, 64, 8, 1)), 1 << (v.bit_length() - 1))
    v = v // q * q
    return v if v != 3072 else v - q


def draw(rng):
    op = rng.choice(("linear", "linear", "grad", "grad", "clip"))
    if op == "clip":
        while True:
            c = {"op": "clip", "dtype": rng.choice(("f32", "f16", "bf16")), "tensors": _log_int(rng, 1, 60), "adapters": _log_int(rng, 1, 64),
                 "rank": _log_int(rng, 1, 64), "K": _width(rng, 64, 2624), "N": _width(rng, 2, 5248),
                 "norm": rng.choice((0.1, 1.0, 1e6))}
            if _elements(c) * (2 if c["dtype"] == "f32" else 1) <= _MOST_ELEMENTS:
                return c
    while True:
        c = {"op": op, "dtype": rng.choice(("f16", "bf16")), "rows": _log_int(rng, 1, 69135), "requests": 0,
             "adapters": _log_int(rng, 1, 64), "rank": _log_int(rng, 1, 64), "K": _width(rng, 64, 2624), "N": _width(rng, 2, 5248),
             "bare": rng.choice((0.0, 0.125, 0.5)), "bias": op == "linear" and rng.random() < 0.5}
        c["requests"] = _log_int(rng, 1, min(256, c["rows"]))
        if c["rows"] * c["K"] * c["N"] <= _MOST_MKN:
            return c


def _elements(c):
    """Gradient elements of a clip case: tensors alternate between A's and B's shapes."""
    n = c["tensors"]
    return c["adapters"] * c["rank"] * (((n + 1) // 2) * c["K"] + (n // 2) * c["N"])


def _requests(case, seed):
    """Row ranges of the requests and the adapter of each (-1: none), from the seed alone."""
    rng = random.Random(seed * 7919 + case["rows"])
    n, T = case["requests"], case["rows"]
    weight = [rng.uniform(0.07, 1.0) for _ in range(n)]
    total, at, cu = sum(weight), 0.0, [0]
    for w in weight:
        at += w
        cu.append(min(T, int(round(T * at / total))))
    cu[-1] = T
    adapter = [rng.randrange(case["adapters"]) for _ in range(n)]
    for i in rng.sample(range(n), int(n * case["bare"])):
        adapter[i] = -1
    return cu, adapter


def _inputs(case, seed):
    dt = _TYPES[case["dtype"]]
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std).to(dtype)

    if case["op"] == "clip":
        spread = random.Random(seed)
        grads = []
        for i in range(case["tensors"]):
            width = case["K"] if i % 2 == 0 else case["N"]
            grads.append(normal(case["adapters"], case["rank"], width, std=1e-3 * math.exp(spread.uniform(-2.0, 2.0))))
        return {"grads": grads}
    T, K, N, n, r = case["rows"], case["K"], case["N"], case["adapters"], case["rank"]
    s = {"x": normal(T, K),  # normalised activations
         "w": normal(N, K, std=0.02),
         "a": normal(n, r, K, std=K ** -0.5),
         "b": normal(n, r, N, std=0.02),  # trained: no longer zero
         "scales": torch.rand(n, generator=g, device="cuda") * 1.5 + 0.5,  # alpha / r
         "bias": normal(N, std=0.1) if case["bias"] else None}
    if case["op"] == "grad":
        s["dy"] = normal(T, N, std=0.05)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] != "clip":
        cu, adapter = _requests(case, seed)
    if not own:
        s["op"] = case["op"]
        if case["op"] == "clip":
            s["norm"] = case["norm"]
            return s
        rows = {}  # what a program keeps of its batch: the rows of each adapter
        for i, a in enumerate(adapter):
            if a >= 0 and cu[i] < cu[i + 1]:
                rows.setdefault(a, []).append(torch.arange(cu[i], cu[i + 1]))
        s["rows"] = [(a, torch.cat(rows[a]).cuda()) for a in sorted(rows)]
        few = case["rows"] <= 8 * len(rows) and case["rows"] * case["rank"] * (case["K"] + case["N"]) <= 1 << 23
        s["each"] = None
        if few and rows:
            of = [(t, a) for i, a in enumerate(adapter) if a >= 0 for t in range(cu[i], cu[i + 1])]
            s["each"] = tuple(torch.tensor(v).cuda() for v in zip(*of))
        return s
    import numpy as np

    from laya_js_b200 import createCudaBackend
    from laya_js_b200 import adapters as ad
    from laya_js_b200 import interop
    b = createCudaBackend(0)
    interop.useTorchStream(b)
    d = {"op": case["op"], "backend": b, "torch": s, "ad": ad, "interop": interop}
    if case["op"] == "clip":
        d["grads"] = [interop.fromTorch(b, t) for t in s["grads"]]
        d["norm"] = case["norm"]
        return d
    for k, v in s.items():
        d[k] = None if v is None else interop.fromTorch(b, v)
    d["plan"] = ad.AdapterPlan(b, np.asarray(cu, np.int32), np.asarray(adapter, np.int32), case["adapters"])
    return d


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    b, ad, interop = s["backend"], s["ad"], s["interop"]
    interop.useTorchStream(b)
    if s["op"] == "linear":
        return interop.toTorch(b, ad.adapter_linear(b, s["x"], s["w"], s["bias"], s["a"], s["b"], s["scales"], s["plan"]))
    if s["op"] == "grad":
        dx, da, db = ad.adapter_linear_grad(b, s["dy"], s["x"], s["w"], s["a"], s["b"], s["scales"], s["plan"])
        return {"dx": interop.toTorch(b, dx), "da": interop.toTorch(b, da), "db": interop.toTorch(b, db)}
    clipped, norm = ad.clip_grad_norm(b, s["grads"], s["norm"])
    return {"grads": [interop.toTorch(b, t) for t in clipped], "norm": interop.toTorch(b, norm)}


def _run_plain(s):
    if s["op"] == "clip":
        total = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
        factor = torch.clamp(s["norm"] / (total + _EPS), max=1.0)
        return {"grads": [(g.float() * factor).to(g.dtype) for g in s["grads"]], "norm": total}
    x, w, dt = s["x"].float(), s["w"].float(), s["x"].dtype
    if s["op"] == "linear":
        y = x @ w.t()
        if s["bias"] is not None:
            y += s["bias"].float()
        if s["each"] is not None:  # few rows: every row's own adapter gathered, rather than a loop over adapters
            rows, of = s["each"]
            u = torch.bmm(s["a"][of].float(), x[rows].unsqueeze(2))
            y[rows] += s["scales"][of, None] * torch.bmm(u.transpose(1, 2), s["b"][of].float()).squeeze(1)
            return y.to(dt)
        for a, rows in s["rows"]:
            u = x[rows] @ s["a"][a].float().t()
            y[rows] += s["scales"][a] * (u @ s["b"][a].float())
        return y.to(dt)
    dy = s["dy"].float()
    dx = dy @ w
    da = torch.zeros(s["a"].shape, device=x.device)
    db = torch.zeros(s["b"].shape, device=x.device)
    for a, rows in s["rows"]:
        xa, dya, down, up = x[rows], dy[rows], s["a"][a].float(), s["b"][a].float()
        g = s["scales"][a] * (dya @ up.t())
        u = s["scales"][a] * (xa @ down.t())
        dx[rows] += g @ down
        da[a] = g.t() @ xa
        db[a] = u.t() @ dya
    return {"dx": dx.to(dt), "da": da.to(dt), "db": db.to(dt)}


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "clip":
        n = _elements(case)
        return {"bytes": 2 * n * size + 4, "flops": 3 * n}
    T, K, N, n, r = case["rows"], case["K"], case["N"], case["adapters"], case["rank"]
    rows = T * (1 - case["bare"])  # rows that have an adapter, about
    banks = n * r * (K + N) * size + 4 * n
    if case["op"] == "linear":
        return {"bytes": (T * K + N * K + T * N + (N if case["bias"] else 0)) * size + banks,
                "flops": 2 * T * K * N + 2 * rows * r * (K + N)}
    # dx = dy·W + g·A;  g = s·dy·Bᵀ, u = s·x·Aᵀ, dA = gᵀ·x, dB = uᵀ·dy
    return {"bytes": (T * N + T * K + N * K + T * K) * size + 2 * banks,
            "flops": 2 * T * K * N + 2 * rows * r * (3 * K + 2 * N)}


def exact(case, seed):
    """The definition in 64 bits, request by request."""
    if not torch.cuda.is_available():
        return None
    s = _inputs(case, seed)
    if case["op"] == "clip":
        g64 = [g.double() for g in s["grads"]]
        norm = math.sqrt(sum(float(torch.dot(g.flatten(), g.flatten())) for g in g64))
        ratio = min(1.0, case["norm"] / (norm + _EPS))
        return {"grads": [g.mul_(ratio) for g in g64], "norm": torch.tensor(norm, dtype=torch.float64)}
    cu, adapter = _requests(case, seed)
    x, w = s["x"].double(), s["w"].double()
    a64, b64, scale = s["a"].double(), s["b"].double(), s["scales"].double()
    spans = [(cu[i], cu[i + 1], adapter[i]) for i in range(len(adapter)) if cu[i + 1] > cu[i]]
    if case["op"] == "linear":
        y = torch.empty((case["rows"], case["N"]), dtype=torch.float64, device="cuda")
        for lo, hi, k in spans:
            # the adapted weight of this request: W + s·Bᵀ·A
            wk = w if k < 0 else torch.addmm(w, b64[k].t(), a64[k], alpha=float(scale[k]))
            torch.matmul(x[lo:hi], wk.t(), out=y[lo:hi])
        if s["bias"] is not None:
            y += s["bias"].double()
        return y
    dy = s["dy"].double()
    dx = torch.empty_like(x)
    da, db = torch.zeros_like(a64), torch.zeros_like(b64)
    for lo, hi, k in spans:
        if k < 0:
            torch.matmul(dy[lo:hi], w, out=dx[lo:hi])
            continue
        sk = float(scale[k])
        torch.matmul(dy[lo:hi], torch.addmm(w, b64[k].t(), a64[k], alpha=sk), out=dx[lo:hi])
        outer = sk * (dy[lo:hi].t() @ x[lo:hi])  # d loss / d (Bᵀ·A), [N, K]
        da[k] += b64[k] @ outer
        db[k] += a64[k] @ outer.t()
    return {"dx": dx, "da": da, "db": db}

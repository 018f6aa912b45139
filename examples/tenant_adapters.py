"""Adapters of many tenants beside one shared encoder: train, then serve.

A frozen ModernBERT-shaped encoder gives every prompt a feature row (its
[CLS] token). Each tenant has its own classification task and its own
low-rank adapters beside a shared two-layer head

    h = relu(dense(f)),  logits = out(h)

Training runs all tenants in one batch: adapter_linear forward, softmax
cross-entropy, adapter_linear_grad back through both layers, clip_grad_norm
over all four adapter gradients, and a plain gradient step on f32 masters.
Serving runs a mixed batch, one row per request, and the encoder itself with
adapters on its projections.

    python examples/tenant_adapters.py [--steps 60]

Synthetic data and random weights; needs a B200.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from laya_js_b200 import createCudaBackend  # noqa: E402
from laya_js_b200 import adapters as ad  # noqa: E402
from laya_js_b200 import workloads as WL  # noqa: E402
from laya_js_b200.host import HostTensor, to_f32  # noqa: E402
from laya_js_b200.modernbert import loadModernBert, parseModernBertConfig  # noqa: E402

DTYPE = "bf16"
CONFIG = {**WL.BASE, "vocab_size": 512, "num_hidden_layers": 2}
TENANTS, PROMPTS, LENGTH, CLASSES, RANK, SCALE = 6, 16, 24, 4, 8, 2.0


def features(b, encoder, ids, mask):
    """The [CLS] rows of the frozen encoder, [prompts, H]."""
    n, length = ids.shape
    hidden = encoder.forward(ids, mask, n, length)
    cls = b.reshape(b.slice(hidden, [0, 0], [n, 1]), [n, hidden.shape[2]])
    rows = b.cast(cls, DTYPE)
    b.dispose(hidden)
    return rows


class TenantHead:
    """The shared head (frozen) and every tenant's adapters beside its two layers."""

    def __init__(self, b, hidden: int, rng):
        self.b = b
        up = lambda a: b.fromHost(ad._host(DTYPE, a))
        self.dense = up(rng.standard_normal((hidden, hidden)) * hidden ** -0.5)
        self.out = up(rng.standard_normal((CLASSES, hidden)) * hidden ** -0.5)
        self.scales = b.fromHost(HostTensor("f32", (TENANTS,), np.full(TENANTS, SCALE, np.float32)))
        f32 = lambda a: b.fromHost(HostTensor("f32", a.shape, a.astype(np.float32)))
        # down-projections random, up-projections zero: training starts from the shared head
        self.masters = [f32(rng.standard_normal((TENANTS, RANK, hidden)) * hidden ** -0.5), f32(np.zeros((TENANTS, RANK, hidden))),
                        f32(rng.standard_normal((TENANTS, RANK, hidden)) * hidden ** -0.5), f32(np.zeros((TENANTS, RANK, CLASSES)))]
        self.params = [b.cast(m, DTYPE) for m in self.masters]

    def forward(self, rows, plan):
        """(dense output, relu of it, logits)."""
        b, (a1, b1, a2, b2) = self.b, self.params
        z = ad.adapter_linear(b, rows, self.dense, None, a1, b1, self.scales, plan)
        h = b.relu(z)
        return z, h, ad.adapter_linear(b, h, self.out, None, a2, b2, self.scales, plan)

    def step(self, rows, onehot, plan, lr: float, max_norm: float):
        """One training step; returns (loss, gradient norm)."""
        b, (a1, b1, a2, b2) = self.b, self.params

        def run():
            z, h, logits = self.forward(rows, plan)
            p = b.softmax(b.cast(logits, "f32"), 1)
            loss = b.scale(b.sum(b.mul(onehot, b.log(p)), 1), -1.0)
            dlogits = b.cast(b.scale(b.sub(p, onehot), 1.0 / rows.shape[0]), DTYPE)
            dh, da2, db2 = ad.adapter_linear_grad(b, dlogits, h, self.out, a2, b2, self.scales, plan)
            dz = b.mul(dh, b.cast(b.greater(z, b.scale(z, 0.0)), DTYPE))
            _, da1, db1 = ad.adapter_linear_grad(b, dz, rows, self.dense, a1, b1, self.scales, plan, want=("da", "db"))
            grads, norm = ad.clip_grad_norm(b, [da1, db1, da2, db2], max_norm)
            masters = [b.sub(m, b.scale(b.cast(g, "f32"), lr)) for m, g in zip(self.masters, grads)]
            return [loss, norm, *masters, *[b.cast(m, DTYPE) for m in masters]]

        loss, norm, *new = b.scope(run)
        for t in (*self.masters, *self.params):
            b.dispose(t)
        self.masters, self.params = new[:4], new[4:]
        value = float(np.mean(b.read(loss).data)), float(b.read(norm).data)
        b.dispose(loss)
        b.dispose(norm)
        return value

    def dispose(self) -> None:
        for t in (self.dense, self.out, self.scales, *self.masters, *self.params):
            self.b.dispose(t)


def main(steps: int = 60, verbose: bool = True) -> dict:
    b = createCudaBackend(0)
    rng = np.random.default_rng(0)
    encoder = loadModernBert(b, parseModernBertConfig(CONFIG), WL.host_getter(WL.random_weights(CONFIG, seed=1)), "f16")
    n, H = TENANTS * PROMPTS, CONFIG["hidden_size"]
    ids = rng.integers(5, CONFIG["vocab_size"], size=(n, LENGTH)).astype(np.int32)
    rows = features(b, encoder, ids, np.ones((n, LENGTH), np.uint8))
    # tenants label the same features differently
    labels = np.stack([rng.integers(0, CLASSES, size=PROMPTS) for _ in range(TENANTS)]).reshape(-1)
    onehot = b.fromHost(HostTensor("f32", (n, CLASSES), np.eye(CLASSES, dtype=np.float32)[labels]))
    plan = ad.AdapterPlan(b, np.arange(TENANTS + 1) * PROMPTS, np.arange(TENANTS), TENANTS)
    head = TenantHead(b, H, rng)
    history = [head.step(rows, onehot, plan, lr=0.5, max_norm=1.0) for _ in range(steps)]
    if verbose:
        for i in range(0, steps, max(1, steps // 6)):
            print(f"step {i:3d}: loss {history[i][0]:.4f}, gradient norm {history[i][1]:.3f}")
        print(f"step {steps - 1:3d}: loss {history[-1][0]:.4f}")

    # serve: the same requests in another order, one row each, every tenant mixed
    order = rng.permutation(n)
    f = b.read(rows)
    mixed = b.fromHost(HostTensor(DTYPE, f.shape, np.ascontiguousarray(f.data[order])))
    each = ad.AdapterPlan(b, np.arange(n + 1), order // PROMPTS, TENANTS)
    trained = to_f32(b.read(head.forward(rows, plan)[2]))
    served = to_f32(b.read(head.forward(mixed, each)[2]))
    accuracy = float(np.mean(served.argmax(1) == labels[order]))
    if verbose:
        print(f"served {n} mixed requests: accuracy {accuracy:.2f}, largest difference from the training batch "
              f"{np.abs(served - trained[order]).max():.2e}")

    # and the encoder itself, with an adapter of each prompt's tenant on its q/k/v and output projections
    bank = lambda out: ad.AdapterBank(b, rng.standard_normal((TENANTS, RANK, H)) * H ** -0.5, rng.standard_normal((TENANTS, out, RANK)) * 0.02,
                                      np.full(TENANTS, SCALE), "f16")
    adapted = ad.EncoderAdapters([{"Wqkv": bank(3 * H), "Wo": bank(H)} for _ in range(CONFIG["num_hidden_layers"])])
    tenants = adapted.batch([0, 1, -1, TENANTS - 1], LENGTH)
    hidden = to_f32(b.read(encoder.forward(ids[:4], np.ones((4, LENGTH), np.uint8), 4, LENGTH, tenants=tenants)))
    plain = to_f32(b.read(encoder.forward(ids[:4], np.ones((4, LENGTH), np.uint8), 4, LENGTH)))
    moved = [float(np.abs(hidden[i] - plain[i]).max()) for i in range(4)]
    if verbose:
        print("encoder with tenants 0, 1, none, 5: hidden rows moved by " + ", ".join(f"{m:.3f}" for m in moved))
    tenants.free()
    adapted.dispose()
    head.dispose()
    encoder.dispose()
    plan.free()
    each.free()
    return {"history": history, "served": served, "trained": trained[order], "accuracy": accuracy, "moved": moved}


if __name__ == "__main__":
    p = argparse.ArgumentParser()
    p.add_argument("--steps", type=int, default=60)
    main(p.parse_args().steps)

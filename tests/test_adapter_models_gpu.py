"""Adapters in use: the encoder with an adapter of each prompt's tenant on its
projections against the oracle with that tenant's weights merged, packed
weights included, and the training example."""
from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import pytest

from adapters_ref import mk, vals
from gpu_util import backend
from laya_js_b200 import adapters as A
from laya_js_b200 import workloads as WL
from laya_js_b200.host import HostTensor, to_f32, unpack_quantized
from laya_js_b200.modernbert import loadModernBert, parseModernBertConfig
from oracle import models as M

pytestmark = pytest.mark.gpu

CFG = {"vocab_size": 512, "hidden_size": 128, "intermediate_size": 192, "num_hidden_layers": 3, "num_attention_heads": 2, "local_attention": 16}
H, I = 128, 192
SHAPES = {"Wqkv": ("attn.Wqkv", 3 * H, H), "Wo": ("attn.Wo", H, H), "Wi": ("mlp.Wi", 2 * I, H), "WoMlp": ("mlp.Wo", H, I)}


def _adapters(b, rng, n, r, dtype, names=A.PROJECTIONS):
    """(EncoderAdapters, merged(W, tenant) -> W with that tenant's adapters, in the values the device holds)."""
    raw = [{k: (rng.standard_normal((n, r, SHAPES[k][2])) * 0.1, rng.standard_normal((n, SHAPES[k][1], r)) * 0.1, rng.uniform(0.5, 2, n))
            for k in names} for _ in range(CFG["num_hidden_layers"])]
    banks = [{k: A.AdapterBank(b, *v, dtype) for k, v in layer.items()} for layer in raw]

    def merged(W, t):
        W = dict(W)
        if t < 0:
            return W
        for i, layer in enumerate(raw):
            for k, (down, up, s) in layer.items():
                d, u = vals(mk(dtype, down[t])), vals(mk(dtype, up[t]))
                key = f"encoder.layers.{i}.{SHAPES[k][0]}.weight"
                W[key] = (W[key] + np.float32(s[t]) * (u @ d)).astype(np.float32)
        return W
    return A.EncoderAdapters(banks), merged


@pytest.mark.parametrize("dtype,quant,tol", [("f32", 0, 1e-4), ("f16", 0, 5e-2), ("f16", 8, 5e-2)])
def test_encoder_with_tenants_matches_merged_weights(dtype, quant, tol):
    """f32: the oracle's own stage tolerance of 1e-5 per stage over three
    layers and four projections each; f16: the encoder tests' 5e-2."""
    b = backend()
    rng = np.random.default_rng(2)
    W = WL.random_weights(CFG, seed=5, norm_std=0.05)
    get = WL.host_getter(W, quant, 64) if quant else WL.host_getter(W)
    enc = loadModernBert(b, parseModernBertConfig(CFG), get, dtype)
    Wf = {k: (unpack_dequantized(get(k)) if quant and hasattr(get(k), "bits") else v.astype(np.float32)) for k, v in W.items()}
    ad, merged = _adapters(b, rng, 4, 8, dtype)
    B, L = 5, 40
    ids = rng.integers(5, 512, size=(B, L)).astype(np.int32)
    valid = np.ones((B, L), np.uint8)
    valid[1, 31:] = 0
    who = [2, 0, -1, 3, 2]
    tenants = ad.batch(who, L)
    got = to_f32(b.read(enc.forward(ids, valid, B, L, tenants=tenants)))
    cfg = M.parse_config(CFG)
    for i, t in enumerate(who):
        want = M.encoder_forward(cfg, merged(Wf, t), ids[i:i + 1], valid[i:i + 1].astype(bool))[0]
        err = np.abs(got[i] - want)[valid[i].astype(bool)].max()
        assert err < tol, f"prompt {i} (tenant {t}): {err}"
    plain = to_f32(b.read(enc.forward(ids, valid, B, L)))
    assert np.abs(got[2] - plain[2]).max() < tol  # the prompt without a tenant
    tenants.free()
    ad.dispose()
    enc.dispose()


def unpack_dequantized(h):
    q = unpack_quantized(h).astype(np.float64)
    N, K = h.shape
    g = np.arange(K) // h.groupSize
    v = q.reshape(N, K) * to_f32(h.scales).astype(np.float64)[:, g]
    return (v + to_f32(h.biases).astype(np.float64)[:, g] if h.biases is not None else v).astype(np.float32)


def test_encoder_adapters_refuse():
    b = backend()
    rng = np.random.default_rng(3)
    bank = lambda n: A.AdapterBank(b, rng.standard_normal((n, 4, H)), rng.standard_normal((n, H, 4)), np.ones(n), "f16")
    two, three = bank(2), bank(3)
    with pytest.raises(ValueError, match="same number"):
        A.EncoderAdapters([{"Wo": two}, {"Wo": three}])
    with pytest.raises(ValueError, match="unknown projections"):
        A.EncoderAdapters([{"Wx": two}])
    with pytest.raises(ValueError, match="AdapterBank"):
        A.AdapterBank(b, np.zeros((2, 4, H)), np.zeros((2, H, 5)), np.ones(2), "f16")
    two.dispose()
    three.dispose()


def test_training_example():
    sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))
    import tenant_adapters
    out = tenant_adapters.main(steps=60, verbose=False)
    losses = [l for l, _ in out["history"]]
    assert losses[-1] < 0.5 * losses[0] and out["accuracy"] > 0.9
    # rows alone against rows in blocks: one bf16 rounding of the hidden layer and one of the logits apart
    assert np.abs(out["served"] - out["trained"]).max() <= 2.0 ** -5 * np.abs(out["trained"]).max()
    assert out["moved"][2] < 1e-2 and min(out["moved"][0], out["moved"][1], out["moved"][3]) > 1e-2

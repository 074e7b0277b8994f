"""EXPERT_CACHE_MOE=1 on the GPU: armed layers that compute their served steps with ops.Experts
over the slots, step after step with experts moving in and out, eager and captured, against the
layer's formula over the full experts in 64 bits (tolerances as in test_gpu_ops.py)."""
from __future__ import annotations

import types

import numpy as np
import pytest
import torch

import gpu_util as gu
from test_generic import new_log, quant_config
from test_gpu_ops import _close, _gen, _moe, _weights
from vllm_expert_cache import ops
from vllm_expert_cache.backends import generic

pytestmark = pytest.mark.gpu

DEV = gu.DEV
E, S, H, I, K = 24, 8, 256, 128, 2
BF16, I8, E4 = torch.bfloat16, torch.int8, torch.float8_e4m3fn
NAMES = {I8: ("w13_weight_scale", "w2_weight_scale"),
         E4: ("w13_weight_scale_inv", "w2_weight_scale_inv")}


class Method:
    """A FusedMoEMethodBase stand-in whose own apply marks the steps that reach it."""

    is_monolithic = False

    def __init__(self, layer, names):
        self.names, self.stock = names, 0
        self.moe_quant_config = self.get_fused_moe_quant_config(layer)
        self.moe_kernel = types.SimpleNamespace(
            fused_experts=types.SimpleNamespace(quant_config=self.moe_quant_config))

    def get_fused_moe_quant_config(self, layer):
        return quant_config(*[getattr(layer, n) for n in self.names])

    def apply(self, layer, x, topk_weights, topk_ids, shared_experts=None,
              shared_experts_input=None):
        self.stock += 1
        return torch.zeros_like(x)


def _layer(monkeypatch, kind):
    monkeypatch.setenv("EXPERT_CACHE_SLOTS", str(S))
    monkeypatch.setenv("EXPERT_CACHE_MOE", "1")
    g = _gen(31)
    # 16-byte slabs of block scales: four blocks a matrix
    h, i = (512, 256) if kind == E4 else (H, I)
    w13, s13 = _weights(g, E, 2 * i, h, kind)
    w2, s2 = _weights(g, E, h, i, kind)
    layer = torch.nn.Module()
    names = NAMES.get(kind, ())
    for name, t in zip(("w13_weight", "w2_weight") + tuple(names), (w13, w2, s13, s2)):
        layer.register_parameter(name, torch.nn.Parameter(t, requires_grad=False))
    layer.global_num_experts, layer.expert_map = E, None
    method = Method(layer, names)
    log = new_log("moe")
    assert generic.arm(layer, method, log.logger)
    assert not log.has("computes its own")
    return layer, method, ops.Experts(w13, w2, s13, s2), h


def _step(rng, tokens, h):
    ids = np.stack([rng.choice(E, K, replace=False) for _ in range(tokens)]).astype(np.int32)
    weights = rng.random((tokens, K), dtype=np.float32) + 0.1
    return (torch.as_tensor(rng.standard_normal((tokens, h), dtype=np.float32), device=DEV).to(BF16),
            torch.as_tensor(weights, device=DEV), torch.as_tensor(ids, device=DEV))


@pytest.mark.parametrize("kind", [BF16, I8, E4], ids=["bf16", "int8", "e4m3"])
def test_served_steps_equal_the_formula(monkeypatch, kind):
    layer, method, whole, h = _layer(monkeypatch, kind)
    rng = np.random.default_rng(5)
    for t in range(24):
        x, weights, ids = _step(rng, int(rng.integers(1, S // K + 1)), h)
        _close(method.apply(layer, x, weights, ids), *_moe(whole, x, weights, ids))
    assert method.stock == 0
    x, weights, ids = _step(rng, S // K + 1, h)       # more ids than slots: read through
    method.apply(layer, x, weights, ids)
    assert method.stock == 1


def test_captured_served_steps_equal_the_formula(monkeypatch):
    layer, method, whole, h = _layer(monkeypatch, BF16)
    rng = np.random.default_rng(6)
    x, weights, ids = _step(rng, 2, h)
    method.apply(layer, x, weights, ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = method.apply(layer, x, weights, ids)
    for t in range(12):
        for static, new in zip((x, weights, ids), _step(rng, 2, h)):
            static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        _close(out, *_moe(whole, x, weights, ids))
    assert method.stock == 0

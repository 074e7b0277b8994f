"""EXPERT_CACHE_MOE=1: which armed layers compute their served steps with ops.Experts, and which
steps. On the CPU against stand-ins; the operator itself is covered by the GPU tests."""
from __future__ import annotations

import types

import pytest
import torch

from test_generic import HID, INTER, E, MoEMethod, S, armed, moe_layer
from vllm_expert_cache import ops
from vllm_expert_cache.backends import generic

H, I = 32, 16


def layer_of(dtype=torch.bfloat16, scales=(), hidden=H, inter=I, **attrs):
    layer = torch.nn.Module()
    for name, shape in (("w13_weight", (E, 2 * inter, hidden)), ("w2_weight", (E, hidden, inter))):
        w = torch.nn.Parameter(torch.zeros(shape).to(dtype), requires_grad=False)
        layer.register_parameter(name, w)
    for name, shape in scales:
        layer.register_parameter(name, torch.nn.Parameter(torch.ones(shape), requires_grad=False))
    layer.global_num_experts, layer.expert_map = E, None
    for name, value in attrs.items():
        setattr(layer, name, value)
    return layer


ROW_SCALES = (("w13_weight_scale", (E, 2 * I, 1)), ("w2_weight_scale", (E, H, 1)))
BLOCK_SCALES = (("w13_weight_scale_inv", (E, 4, 4)), ("w2_weight_scale_inv", (E, 4, 2)))


@pytest.fixture(autouse=True)
def own_experts(monkeypatch):
    """The operator's checks without a device, and its calls recorded."""
    monkeypatch.setenv("EXPERT_CACHE_SLOTS", str(S))
    monkeypatch.setenv("EXPERT_CACHE_MOE", "1")
    monkeypatch.setattr(ops, "_on_gpu", lambda *t: t[0].device)
    calls = []

    def call(self, x, topk_weights, slot_ids, out=None):
        calls.append((self, x, topk_weights, slot_ids))
        return torch.full_like(x, 7.0)

    monkeypatch.setattr(ops.Experts, "__call__", call)
    return calls


def step(method, layer, tokens=1, ids=2, dtype=torch.bfloat16, **kw):
    layer._expert_cache.refresh = lambda i: i.clone()
    return method.apply(layer, torch.randn(tokens, H).to(dtype),
                        kw.pop("weights", torch.ones(tokens, ids)),
                        kw.pop("topk_ids", torch.zeros(tokens, ids, dtype=torch.int32)), **kw)


@pytest.mark.parametrize("dtype,scales,hidden,inter", [
    (torch.bfloat16, (), H, I), (torch.float16, (), H, I), (torch.int8, ROW_SCALES, H, I),
    (torch.float8_e4m3fn, BLOCK_SCALES, 512, 256)], ids=["bf16", "f16", "int8", "e4m3"])
def test_served_steps_are_computed_over_the_slots(own_experts, dtype, scales, hidden, inter):
    layer = layer_of(dtype, scales, hidden, inter)
    method = MoEMethod(layer, [n for n, _ in scales])
    ok, log = armed(layer, method)
    assert ok and not log.has("computes its own")
    layer._expert_cache.refresh = lambda i: i.clone()
    x = torch.randn(1, hidden).to(torch.float16 if dtype == torch.float16 else torch.bfloat16)
    out = method.apply(layer, x, torch.ones(1, 2), torch.zeros(1, 2, dtype=torch.int32))
    assert (out == 7).all() and not method.calls
    experts, got, _, ids = own_experts[0]
    assert got is x and ids.shape == (1, 2)
    cache = layer._expert_cache
    assert experts.w13.data_ptr() == cache.slots["w13_weight"].data_ptr()
    assert experts.w2.data_ptr() == cache.slots["w2_weight"].data_ptr()
    if scales:
        assert experts.w13_scale.data_ptr() == cache.slots[scales[0][0]].data_ptr()
        assert experts.w2_scale.data_ptr() == cache.slots[scales[1][0]].data_ptr()


def test_off_by_default(own_experts, monkeypatch):
    monkeypatch.delenv("EXPERT_CACHE_MOE")
    layer = layer_of()
    method = MoEMethod(layer)
    assert armed(layer, method)[0]
    step(method, layer)
    assert len(method.calls) == 1 and not own_experts


@pytest.mark.parametrize("kw", [
    dict(tokens=3), dict(shared_experts=object()), dict(dtype=torch.float32),
    dict(weights=torch.ones(1, 2, dtype=torch.bfloat16)),
    dict(topk_ids=torch.zeros(1, 2, dtype=torch.int16))],
    ids=["wide", "shared", "f32", "weights", "ids"])
def test_other_steps_go_to_the_stock_kernel(own_experts, kw):
    layer = layer_of()
    method = MoEMethod(layer)
    assert armed(layer, method)[0]
    step(method, layer, **kw)
    assert len(method.calls) == 1 and not own_experts


@pytest.mark.parametrize("x,weights", [(torch.zeros(1, H + 8), torch.ones(1, 2)),
                                       (torch.zeros(1, 1, H), torch.ones(1, 2)),
                                       (torch.zeros(1, H), torch.ones(1, 2, 1))],
                         ids=["padded", "batched", "weights"])
def test_steps_of_other_shapes_go_to_the_stock_kernel(own_experts, x, weights):
    layer = layer_of()
    method = MoEMethod(layer)
    assert armed(layer, method)[0]
    layer._expert_cache.refresh = lambda i: i.clone()
    method.apply(layer, x.bfloat16(), weights, torch.zeros(1, 2, dtype=torch.int32))
    assert len(method.calls) == 1 and not own_experts


@pytest.mark.parametrize("layer,method,reason", [
    (lambda: moe_layer(), lambda l: MoEMethod(l), "float32"),
    (lambda: layer_of(activation="gelu"), lambda l: MoEMethod(l), "gelu"),
    (lambda: layer_of(apply_router_weight_on_input=True), lambda l: MoEMethod(l), "input"),
    (lambda: layer_of(torch.int8), lambda l: MoEMethod(l), "scale"),
    (lambda: layer_of(scales=ROW_SCALES), lambda l: MoEMethod(l, [n for n, _ in ROW_SCALES]),
     "no scales"),
    (lambda: layer_of(torch.int8, ROW_SCALES + (("zp", (E, 4)), ("zp2", (E, 4)))),
     lambda l: MoEMethod(l, ["w13_weight_scale", "w2_weight_scale", "zp", "zp2"]), "zp"),
], ids=["f32", "gelu", "input", "int8", "scaled-bf16", "zero-points"])
def test_layers_that_keep_the_stock_kernel(own_experts, layer, method, reason):
    l = layer()
    m = method(l)
    ok, log = armed(l, m)
    assert ok and log.has("computes its own served steps") and log.has(reason)
    l._expert_cache.refresh = lambda i: i.clone()
    m.apply(l, torch.randn(1, HID), torch.ones(1, 2), torch.zeros(1, 2, dtype=torch.int32))
    assert len(m.calls) == 1 and not own_experts


def test_weights_in_another_kernels_layout_keep_the_stock_kernel(own_experts):
    layer = layer_of()
    layer.w13_weight.is_shuffled = True
    ok, log = armed(layer, MoEMethod(layer))
    assert ok and log.has("layout")


def test_silu_as_an_enum_member_is_taken(own_experts):
    layer = layer_of(activation=types.SimpleNamespace(value="silu"))
    method = MoEMethod(layer)
    assert armed(layer, method)[0]
    step(method, layer)
    assert len(own_experts) == 1


def test_packed_weights_keep_the_stock_kernel(own_experts):
    layer = torch.nn.Module()
    for name, shape in (("w13_weight_packed", (E, INTER, HID)), ("w2_weight_packed", (E, HID, 8))):
        layer.register_parameter(name, torch.nn.Parameter(torch.zeros(shape), requires_grad=False))
    layer.global_num_experts, layer.expert_map = E, None

    class Packed(MoEMethod):
        def apply(self, layer, *args, **kw):
            self.calls.append(args)

    method = Packed(layer)
    ok, log = armed(layer, method)
    assert ok and log.has("packed")
    assert generic.settings.moe


@pytest.mark.parametrize("kw", [dict(x=True), dict(weights=True)], ids=["x", "weights"])
def test_steps_that_need_a_gradient_go_to_the_stock_kernel(own_experts, kw):
    layer = layer_of()
    method = MoEMethod(layer)
    assert armed(layer, method)[0]
    layer._expert_cache.refresh = lambda i: i.clone()
    x, weights = torch.randn(1, H).bfloat16(), torch.ones(1, 2)
    x.requires_grad_("x" in kw)
    weights.requires_grad_("weights" in kw)
    ids = torch.zeros(1, 2, dtype=torch.int32)
    method.apply(layer, x, weights, ids)
    assert len(method.calls) == 1 and not own_experts
    with torch.no_grad():
        method.apply(layer, x, weights, ids)
    assert len(method.calls) == 1 and len(own_experts) == 1

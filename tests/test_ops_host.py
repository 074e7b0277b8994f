"""What the operators (vllm_expert_cache/ops.py and their C entry points) refuse, checked
without a GPU: every refusal comes before any HIP call."""
from __future__ import annotations

import ctypes

import pytest
import torch

from vllm_expert_cache import _lib, ops

BF16, F16, F32, I8, E4 = (torch.bfloat16, torch.float16, torch.float32, torch.int8,
                          torch.float8_e4m3fn)
P = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


# ---- C entry points -----------------------------------------------------------------------

def _route(lib, **over):
    a = dict(logits=0x1000, type=0, stride=8, bias=None, T=2, E=8, k=2, scoring=0, groups=1,
             topk_groups=1, renorm=1, scale=1.0, weights=0x2000, ids=0x3000, id_bytes=4)
    a.update(over)
    return lib.expert_cache_route(*a.values(), None)


@pytest.mark.parametrize("over", [
    dict(T=-1), dict(E=0), dict(E=1025, stride=1025), dict(stride=7), dict(type=3),
    dict(type=-1), dict(k=0), dict(k=9), dict(E=128, stride=128, k=65), dict(scoring=2),
    dict(scoring=-1), dict(groups=0), dict(groups=3), dict(E=130, stride=130, groups=65),
    dict(groups=2, topk_groups=0), dict(groups=2, topk_groups=3),
    dict(groups=4, topk_groups=1, k=3), dict(id_bytes=2), dict(logits=None),
    dict(weights=None), dict(ids=None)], ids=str)
def test_route_rejects(lib, over):
    assert _route(lib, **over) == -1


@pytest.mark.parametrize("over", [
    dict(T=2 ** 21 + 1), dict(T=2 ** 31 - 1, E=1, stride=1, k=1),
    dict(weights=0x1020), dict(ids=0x1038), dict(ids=0x2008), dict(bias=0x2008),
    dict(bias=0x2FF0), dict(type=1, weights=0x101C)], ids=str)
def test_route_rejects_what_meets_or_is_too_long(lib, over):
    assert _route(lib, **over) == -1


@pytest.mark.parametrize("over", [dict(out=0x40008), dict(out=0x50000), dict(ids=0x60030)],
                         ids=str)
def test_results_over_ids_and_weights_are_refused(lib, over):
    assert _moe(lib, **over) == -1


def test_adapters_past_what_a_grid_holds_are_refused(lib):
    assert _adapt(lib, T=2 ** 21 + 1) == -1
    assert _adapt(lib, O=2 ** 21 + 1, bs=2 ** 21 + 1, os=2 ** 21 + 1) == -1


def test_nothing_to_do_is_no_call(lib):
    assert _route(lib, T=0, logits=None, weights=None, ids=None) == 0
    assert _moe(lib, T=0, x=None, out=None, ids=None, work=None) == 0
    assert _adapt(lib, T=0, x=None, base=None, out=None, ids=None, work=None) == 0


def _layer(**over):
    f = dict(S=4, H=32, I=16, type=1, weights=1, w13=0x10000, w2=0x20000, s13=None, s2=None)
    f.update({k: v for k, v in over.items() if k in f})
    return _lib.Experts(*f.values())


def _moe(lib, **over):
    e = _layer(**over)
    a = dict(x=0x30000, xs=32, probs=0x40000, ids=0x50000, id_bytes=4, T=2, k=2, out=0x60000,
             os=32, work=0x70000)
    a.update({k: v for k, v in over.items() if k in a})
    return lib.expert_cache_moe(ctypes.addressof(e), *a.values(), None)


BAD_LAYER = [dict(S=0), dict(H=0), dict(I=0), dict(H=-8), dict(type=0), dict(type=3),
             dict(weights=2), dict(weights=0), dict(weights=5), dict(H=36), dict(I=20),
             dict(weights=3, s13=16, s2=16, H=40), dict(weights=4, s13=16, s2=16, I=24),
             dict(T=-1), dict(k=0), dict(k=65), dict(T=513)]


@pytest.mark.parametrize("over", BAD_LAYER + [
    dict(w13=None), dict(w2=None), dict(w13=0x10008), dict(w2=0x20004),
    dict(weights=3), dict(weights=4, s13=16), dict(weights=3, s2=16),
    dict(weights=3, s13=16, s2=20), dict(weights=4, s13=8, s2=16), dict(x=None),
    dict(x=0x30002), dict(xs=36), dict(xs=24), dict(out=None), dict(os=24), dict(probs=None),
    dict(ids=None), dict(id_bytes=2), dict(work=None), dict(work=0x70008),
    dict(out=0x30000), dict(out=0x30000 + 64), dict(out=0x30000 - 100)], ids=str)
def test_moe_rejects(lib, over):
    assert _moe(lib, **over) == -1


@pytest.mark.parametrize("over", BAD_LAYER, ids=str)
def test_moe_workspace_rejects(lib, over):
    size = ctypes.c_long(-5)
    assert lib.expert_cache_moe_workspace(ctypes.addressof(_layer(**over)), over.get("T", 2),
                                          over.get("k", 2), ctypes.addressof(size)) == -1
    assert size.value == -5


def test_null_handles_are_rejected(lib):
    size = ctypes.c_long()
    at = ctypes.addressof(size)
    assert lib.expert_cache_moe_workspace(None, 1, 1, at) == -1
    assert lib.expert_cache_moe_workspace(ctypes.addressof(_layer()), 1, 1, None) == -1
    assert lib.expert_cache_moe(None, 16, 32, 16, 16, 4, 1, 1, 16, 32, 16, None) == -1
    assert lib.expert_cache_adapt_workspace(None, 1, at) == -1
    assert lib.expert_cache_adapt_workspace(ctypes.addressof(_lora()), 1, None) == -1
    assert lib.expert_cache_adapt(None, 16, 32, 16, 4, 1, 16, 32, 16, 32, 16, None) == -1


def _lora(**over):
    f = dict(S=4, H=32, O=24, R=8, type=1, a=0x10000, b=0x20000, scales=None)
    f.update({k: v for k, v in over.items() if k in f})
    return _lib.Adapters(*f.values())


def _adapt(lib, **over):
    l = _lora(**over)
    a = dict(x=0x30000, xs=32, ids=0x40000, id_bytes=4, T=2, base=0x50000, bs=24, out=0x60000,
             os=24, work=0x70000)
    a.update({k: v for k, v in over.items() if k in a})
    return lib.expert_cache_adapt(ctypes.addressof(l), *a.values(), None)


@pytest.mark.parametrize("over", [
    dict(S=0), dict(H=0), dict(O=0), dict(R=0), dict(H=36), dict(R=12), dict(R=264),
    dict(type=0), dict(type=3), dict(T=-1), dict(a=None), dict(b=None), dict(a=0x10002),
    dict(b=0x20008), dict(x=None), dict(x=0x30004), dict(xs=33), dict(xs=24), dict(ids=None),
    dict(id_bytes=1), dict(base=None), dict(bs=16), dict(out=None), dict(os=16),
    dict(work=None), dict(work=0x70004),
    dict(out=0x50000, os=32),            # base's address at another stride
    dict(out=0x50002), dict(out=0x50000 - 2), dict(out=0x30000),
], ids=str)
def test_adapt_rejects(lib, over):
    assert _adapt(lib, **over) == -1


@pytest.mark.parametrize("over", [dict(S=0), dict(H=4), dict(R=264), dict(type=0), dict(T=-1)],
                         ids=str)
def test_adapt_workspace_rejects(lib, over):
    size = ctypes.c_long()
    assert lib.expert_cache_adapt_workspace(ctypes.addressof(_lora(**over)), over.get("T", 2),
                                            ctypes.addressof(size)) == -1


def test_workspaces_cover_what_is_written(lib):
    """Hidden values (two bfloat16) and outputs a pair; low-rank values a token."""
    size = ctypes.c_long()
    for T, k, H, I in ((1, 1, 32, 16), (16, 64, 64, 128), (1024, 1, 8, 8)):
        e = _layer(H=H, I=I)
        assert lib.expert_cache_moe_workspace(ctypes.addressof(e), T, k,
                                              ctypes.addressof(size)) == 0
        assert size.value >= T * k * 4 * I
    for T, H, R in ((1, 32, 8), (1, 65536, 256), (5000, 4096, 64)):
        l = _lora(H=H, R=R)
        assert lib.expert_cache_adapt_workspace(ctypes.addressof(l), T,
                                                ctypes.addressof(size)) == 0
        assert size.value >= 4 * T * R

@pytest.mark.parametrize("H,rows", [(32, 8), (2048, 8), (2064, 16), (2816, 16), (4080, 16),
                                    (4096, 16), (4112, 8), (6144, 8), (6160, 16), (8192, 16),
                                    (8208, 8), (14336, 8)])
def test_rows_of_a_workgroup_down(lib, H, rows):
    """Down projections of a few tokens: 16 rows a workgroup, or 8 where the fullest of 256 compute
    units then has fewer rows. The workspace has a counter of 4 bytes a workgroup (and, where
    several share their rows, 16 x rows floats each)."""
    fullest = {r: -(-(-(-H // r)) // 256) * r for r in (8, 16)}
    assert rows == (8 if fullest[8] < fullest[16] else 16)
    size = ctypes.c_long()
    e = _layer(H=H, I=16)
    assert lib.expert_cache_moe_workspace(ctypes.addressof(e), 1, 1, ctypes.addressof(size)) == 0
    groups = -(-H // rows)
    assert size.value == 4 * 16 + 64 * rows * groups + 48 + 4 * groups


# ---- Python -------------------------------------------------------------------------------

@pytest.fixture
def anywhere(monkeypatch):
    """Lets CPU tensors past the device check, so that the checks after it are reached."""
    monkeypatch.setattr(ops, "_on_gpu", lambda *t: t[0].device)


def test_tensors_on_the_host_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        ops.route(torch.zeros(2, 8), 2)
    with pytest.raises(ValueError, match="GPU"):
        ops.Experts(torch.zeros(2, 32, 16, dtype=BF16), torch.zeros(2, 16, 16, dtype=BF16))
    with pytest.raises(ValueError, match="GPU"):
        ops.Adapters(torch.zeros(2, 8, 16, dtype=BF16), torch.zeros(2, 16, 8, dtype=BF16))


@pytest.mark.parametrize("logits,kw", [
    (torch.zeros(8), {}), (torch.zeros(2, 8, dtype=torch.float64), {}),
    (torch.zeros(2, 1025), {}), (torch.zeros(2, 0), {}),
    (torch.zeros(2, 8), dict(scoring="tanh")), (torch.zeros(2, 8), dict(id_dtype=torch.int16)),
    (torch.zeros(2, 8), dict(groups=3)), (torch.zeros(2, 8), dict(groups=2, topk_groups=3)),
    (torch.zeros(2, 8), dict(top_k=9)), (torch.zeros(2, 8), dict(top_k=0)),
    (torch.zeros(2, 8), dict(groups=4, top_k=3)), (torch.zeros(2, 100), dict(top_k=65)),
    (torch.zeros(2, 8), dict(bias=torch.zeros(7))),
    (torch.zeros(2, 8), dict(bias=torch.zeros(8, dtype=BF16))),
    (torch.zeros(2, 8), dict(bias=torch.zeros(16)[::2]))])
def test_route_arguments(logits, kw):
    with pytest.raises(ValueError) as e:
        ops.route(logits, kw.pop("top_k", 2), **kw)
    assert "GPU" not in str(e.value)


def _w(S=2, H=32, I=16, dtype=BF16):
    return torch.zeros(S, 2 * I, H).to(dtype), torch.zeros(S, H, I).to(dtype)


@pytest.mark.parametrize("make", [
    lambda: ops.Experts(torch.zeros(2, 32, dtype=BF16), _w()[1]),
    lambda: ops.Experts(_w()[0], _w(dtype=F16)[1]),
    lambda: ops.Experts(_w()[0][:, :31], _w()[1]),
    lambda: ops.Experts(_w()[0], _w(S=3)[1]),
    lambda: ops.Experts(_w()[0], _w(I=24)[1]),
    lambda: ops.Experts(*_w(dtype=F32)),
    lambda: ops.Experts(*_w(dtype=torch.uint8)),
    lambda: ops.Experts(*_w(H=36)),
    lambda: ops.Experts(*_w(I=20)),
    lambda: ops.Experts(*_w(H=40, dtype=I8), torch.ones(2, 32), torch.ones(2, 40)),
    lambda: ops.Experts(*_w(I=24, dtype=I8), torch.ones(2, 48), torch.ones(2, 32)),
    lambda: ops.Experts(_w()[0].transpose(1, 2).contiguous().transpose(1, 2), _w()[1]),
    lambda: ops.Experts(torch.zeros(2 * 32 * 32 + 1, dtype=BF16)[1:].view(2, 32, 32), _w()[1]),
], ids=range(13))
def test_experts_weights(anywhere, make):
    with pytest.raises(ValueError):
        make()


@pytest.mark.parametrize("dtype,s13,s2", [
    (BF16, torch.ones(2, 32), None), (I8, None, None), (I8, torch.ones(2, 32), None),
    (I8, torch.ones(2, 31), torch.ones(2, 32)), (I8, torch.ones(32), torch.ones(2, 32)),
    (I8, torch.ones(2, 32, dtype=BF16), torch.ones(2, 32)),
    (I8, torch.ones(2, 64)[:, ::2], torch.ones(2, 32)),
    (E4, torch.ones(2, 32), torch.ones(2, 32)), (E4, torch.ones(2, 1, 1), torch.ones(2, 1, 2))])
def test_experts_scales(anywhere, dtype, s13, s2):
    with pytest.raises(ValueError):
        ops.Experts(*_w(dtype=dtype), s13, s2)


def test_scales_with_a_trailing_one_are_taken(anywhere):
    ops.Experts(*_w(dtype=I8), torch.ones(2, 32, 1), torch.ones(2, 32, 1))
    ops.Experts(*_w(H=144, dtype=E4), torch.ones(2, 1, 2), torch.ones(2, 2, 1))


def _call(T=3, k=2, H=32, dtype=BF16, ids=torch.int32):
    return [torch.zeros(T, H, dtype=dtype), torch.zeros(T, k), torch.zeros(T, k, dtype=ids)]


@pytest.mark.parametrize("x,p,i,out", [
    (*_call(H=16), None), (*_call(dtype=F16), None), (*_call(dtype=F32), None),
    (*_call(ids=torch.int16), None), (*_call(T=600), None), (*_call(T=1, k=65), None),
    (_call()[0], _call(k=3)[1], _call()[2], None), (_call()[0], _call(T=2)[1], _call(T=2)[2], None),
    (_call()[0], _call()[1].to(BF16), _call()[2], None),
    (_call()[0], *[t[0] for t in _call()[1:]], None),
    (*_call(), torch.zeros(3, 32, dtype=F16)), (*_call(), torch.zeros(2, 32, dtype=BF16)),
    (*_call(), torch.zeros(32, 3, dtype=BF16).t()),
    (*_call(), torch.zeros(1, 32, dtype=BF16).expand(3, 32)),
], ids=range(14))
def test_experts_arguments(anywhere, x, p, i, out):
    with pytest.raises(ValueError):
        ops.Experts(*_w())(x, p, i, out)


def _ab(S=2, R=8, H=32, O=24, dtype=BF16):
    return torch.zeros(S, R, H, dtype=dtype), torch.zeros(S, O, R, dtype=dtype)


@pytest.mark.parametrize("make", [
    lambda: ops.Adapters(_ab()[0][0], _ab()[1]), lambda: ops.Adapters(*_ab(dtype=F32)),
    lambda: ops.Adapters(_ab()[0], _ab(dtype=F16)[1]), lambda: ops.Adapters(_ab()[0], _ab(S=3)[1]),
    lambda: ops.Adapters(_ab()[0], _ab(R=16)[1]), lambda: ops.Adapters(*_ab(R=12)),
    lambda: ops.Adapters(*_ab(R=264)), lambda: ops.Adapters(*_ab(H=36)),
    lambda: ops.Adapters(*_ab(O=0)), lambda: ops.Adapters(_ab()[0][:, ::1, :].flip(1)[:, ::2], _ab()[1]),
    lambda: ops.Adapters(_ab(S=4)[0][::2], _ab()[1]),
    lambda: ops.Adapters(*_ab(), torch.ones(3)), lambda: ops.Adapters(*_ab(), torch.ones(2, dtype=BF16)),
], ids=range(13))
def test_adapters_weights(anywhere, make):
    with pytest.raises(ValueError):
        make()


def _rows(T=3, H=32, O=24, dtype=BF16, ids=torch.int32):
    return [torch.zeros(T, H, dtype=dtype), torch.zeros(T, O, dtype=dtype),
            torch.zeros(T, dtype=ids)]


@pytest.mark.parametrize("x,base,ids,out", [
    (*_rows(H=24), None), (*_rows(O=23), None), (*_rows(dtype=F16), None),
    (*_rows(ids=torch.uint8), None), (_rows(T=2)[0], *_rows()[1:], None),
    (*_rows()[:2], _rows(T=4)[2], None), (*_rows()[:2], torch.zeros(3, 1, dtype=torch.int32), None),
    (*_rows(), torch.zeros(3, 24, dtype=F16)), (*_rows(), torch.zeros(24, 3, dtype=BF16).t()),
], ids=range(9))
def test_adapters_arguments(anywhere, x, base, ids, out):
    with pytest.raises(ValueError):
        ops.Adapters(*_ab())(x, base, ids, out)


def test_what_is_too_long_is_refused(anywhere):
    with pytest.raises(ValueError):
        ops.route(torch.empty(ops.MAX_TOKENS + 1, 1), 1)
    with pytest.raises(ValueError):
        ops.Adapters(torch.empty(1, 8, 8, dtype=BF16),
                     torch.empty(1, ops.MAX_OUTPUTS + 1, 8, dtype=BF16))
    with pytest.raises(ValueError):
        ops.Adapters(torch.empty(1, 8, ops.MAX_LENGTH + 8, dtype=BF16),
                     torch.empty(1, 8, 8, dtype=BF16))
    with pytest.raises(ValueError):
        ops.Experts(torch.empty(1, 32, ops.MAX_LENGTH + 16, dtype=I8),
                    torch.empty(1, ops.MAX_LENGTH + 16, 16, dtype=I8))
    T = ops.MAX_TOKENS + 1
    with pytest.raises(ValueError):
        ops.Adapters(*_ab(H=8, O=1))(torch.empty(T, 8, dtype=BF16), torch.empty(T, 1, dtype=BF16),
                                     torch.empty(T, dtype=torch.int32))


@pytest.fixture
def no_kernels(anywhere, monkeypatch):
    """Calls that every check lets through, without a device."""
    calls = []
    monkeypatch.setattr(ops, "_on_device", lambda device, call, *args: calls.append(args) or 0)
    return calls


GRAD_CALLS = {
    "route": (lambda t: ops.route(t["logits"], 2, bias=t["bias"]), ("logits", "bias")),
    "experts": (lambda t: ops.Experts(t["w13"], t["w2"], t["s13"], t["s2"])(t["x"], t["p"], t["i"]),
                ("s13", "s2", "x", "p")),
    "bf16": (lambda t: ops.Experts(t["v13"], t["v2"])(t["x"], t["p"], t["i"], out=t["out"]),
             ("v13", "v2", "x", "p", "out")),
    "adapters": (lambda t: ops.Adapters(t["a"], t["b"], t["f"])(t["x"], t["base"], t["j"]),
                 ("a", "b", "f", "x", "base")),
    "out": (lambda t: ops.Adapters(t["a"], t["b"])(t["x"], t["base"], t["j"], out=t["low"]),
            ("low",)),
}


def _grad_tensors():
    w13, w2 = _w(dtype=I8)
    v13, v2 = _w()
    x, p, i = _call()
    a, b = _ab()
    _, base, j = _rows()
    return dict(logits=torch.zeros(2, 8), bias=torch.zeros(8), w13=w13, w2=w2,
                s13=torch.ones(2, 32), s2=torch.ones(2, 32), v13=v13, v2=v2, x=x, p=p, i=i,
                out=torch.zeros(3, 32, dtype=BF16), a=a, b=b, f=torch.ones(2), base=base, j=j,
                low=torch.zeros(3, 24, dtype=BF16))


@pytest.mark.parametrize("op,name", [(op, n) for op, (_, names) in GRAD_CALLS.items()
                                     for n in names])
def test_what_needs_a_gradient_is_refused(no_kernels, op, name):
    """A result without a graph would leave the gradient out without a word."""
    t = _grad_tensors()
    call = GRAD_CALLS[op][0]
    call(t)
    t[name].requires_grad_()
    with pytest.raises(ValueError, match="backward"):
        call(t)
    assert len(no_kernels) == 1
    with torch.no_grad():
        call(t)
    with torch.inference_mode():
        call(t)
    t[name] = t[name].detach()
    call(t)
    assert len(no_kernels) == 4

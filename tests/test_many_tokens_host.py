"""What the operators for many tokens (vllm_expert_cache/ops.py and their C entry points) refuse,
checked without a GPU: every refusal comes before any HIP call."""
from __future__ import annotations

import ctypes

import pytest
import torch

from vllm_expert_cache import _lib, ops

BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


# ---- C entry points -----------------------------------------------------------------------

def _sort(lib, **over):
    a = dict(ids=0x1000, id_bytes=4, T=4, k=2, S=3, offsets=0x2000, rows=0x3000, places=0x4000,
             work=None)
    a.update(over)
    return lib.expert_cache_sort(*a.values(), None)


@pytest.mark.parametrize("over", [
    dict(T=-1), dict(k=0), dict(k=65), dict(S=0), dict(S=1025), dict(id_bytes=2),
    dict(T=2 ** 24, k=2), dict(T=2 ** 31 - 1, k=64), dict(ids=None), dict(offsets=None),
    dict(rows=None), dict(places=None), dict(T=20000), dict(T=20000, work=0x5008),
    dict(offsets=0x101C), dict(rows=0x101C), dict(places=0x301C), dict(offsets=0x401C),
    dict(ids=0x2FF4, rows=0x3008)], ids=str)
def test_sort_rejects(lib, over):
    assert _sort(lib, **over) == -1


def test_sort_workspace(lib):
    size = ctypes.c_long(-5)
    at = ctypes.addressof(size)
    for T, k, S in ((-1, 1, 1), (1, 0, 1), (1, 65, 1), (1, 1, 0), (1, 1, 1025), (2 ** 24, 2, 1)):
        assert lib.expert_cache_sort_workspace(T, k, S, at) == -1
    assert lib.expert_cache_sort_workspace(1, 1, 1, None) == -1
    assert size.value == -5
    for T, k, S in ((0, 1, 1), (512, 8, 1024)):
        assert lib.expert_cache_sort_workspace(T, k, S, at) == 0 and size.value == 0
    # counts of every key and workgroup, at most 256 of those
    assert lib.expert_cache_sort_workspace(513, 8, 100, at) == 0
    assert size.value == 4 * 5 * 101
    assert lib.expert_cache_sort_workspace(2 ** 24, 1, 1024, at) == 0
    assert size.value == 4 * 256 * 1025


def _dispatch(lib, **over):
    a = dict(x=0x10000, type=1, xs=32, places=0x20000, rows=0x30000, T=4, k=2, H=32,
             out=0x40000, os=32)
    a.update(over)
    return lib.expert_cache_dispatch(*a.values(), None)


@pytest.mark.parametrize("over", [
    dict(T=-1), dict(k=0), dict(k=65), dict(type=-1), dict(type=3), dict(H=0),
    dict(H=2 ** 20 + 1, xs=2 ** 21, os=2 ** 21), dict(xs=31), dict(os=31), dict(x=None),
    dict(places=None), dict(rows=None), dict(out=None), dict(out=0x10000 + 254),
    dict(out=0x20000 + 28), dict(out=0x30000 + 28),
    dict(x=0x40000 + 8 * 64 - 2),
    dict(T=2 ** 24, k=1, H=2 ** 20, xs=2 ** 20, os=2 ** 20)], ids=str)
def test_dispatch_rejects(lib, over):
    assert _dispatch(lib, **over) == -1


def _combine(lib, **over):
    a = dict(y=0x10000, type=1, ys=32, w=0x50000, places=0x20000, T=4, k=2, H=32, out=0x40000,
             os=32)
    a.update(over)
    return lib.expert_cache_combine(*a.values(), None)


@pytest.mark.parametrize("over", [
    dict(T=-1), dict(k=0), dict(k=65), dict(type=-1), dict(type=3), dict(H=0),
    dict(H=2 ** 20 + 1, ys=2 ** 21, os=2 ** 21), dict(ys=31), dict(os=31), dict(y=None),
    dict(places=None), dict(out=None), dict(out=0x10000 + 510), dict(out=0x20000),
    dict(out=0x50000), dict(w=0x40000 + 254)], ids=str)
def test_combine_rejects(lib, over):
    assert _combine(lib, **over) == -1


def _combine_grad(lib, **over):
    a = dict(g=0x10000, type=1, gs=32, y=0x20000, ys=32, w=0x30000, places=0x40000,
             rows=0x50000, T=4, k=2, H=32, dy=0x60000, ds=32, dw=0x70000)
    a.update(over)
    return lib.expert_cache_combine_grad(*a.values(), None)


@pytest.mark.parametrize("over", [
    dict(T=-1), dict(k=0), dict(type=3), dict(H=0), dict(gs=31), dict(ys=31),
    dict(ds=31), dict(g=None), dict(y=None), dict(places=None), dict(rows=None),
    dict(dy=None, dw=None), dict(dy=0x10000), dict(dy=0x20000), dict(dy=0x30000), dict(dy=0x40000),
    dict(dy=0x50000), dict(dy=0x70000), dict(dw=0x10000), dict(dw=0x20000), dict(dw=0x30000),
    dict(dw=0x40000), dict(dw=0x50000), dict(dw=0x60000 + 508)], ids=str)
def test_combine_grad_rejects(lib, over):
    assert _combine_grad(lib, **over) == -1


def _quantize(lib, **over):
    a = dict(x=0x10000, type=1, xs=40, T=4, H=40, q=0x20000, qs=48, scales=0x30000)
    a.update(over)
    return lib.expert_cache_quantize(*a.values(), None)


@pytest.mark.parametrize("over", [
    dict(type=0), dict(type=3), dict(T=-1), dict(T=2 ** 24 + 1), dict(H=0),
    dict(H=2 ** 20 + 1, xs=2 ** 21, qs=2 ** 21), dict(xs=39), dict(qs=32), dict(qs=56),
    dict(x=None), dict(q=None), dict(q=0x20008), dict(scales=None), dict(q=0x10100),
    dict(scales=0x20000 + 188), dict(scales=0x10000)], ids=str)
def test_quantize_rejects(lib, over):
    assert _quantize(lib, **over) == -1


def _linear(lib, **over):
    f = dict(O=24, H=40, ws=48, w=0x10000, scale=0x20000, bias=None)
    f.update({k: v for k, v in over.items() if k in f})
    l = _lib.Linear(*f.values())
    a = dict(x=0x30000, type=1, xs=40, x_scales=None, T=4, out=0x40000, out_type=1, os=24,
             work=0x50000)
    a.update({k: v for k, v in over.items() if k in a})
    return lib.expert_cache_linear8(ctypes.addressof(l), *a.values(), None)


Q = dict(type=3, xs=48, x_scales=0x60000)


@pytest.mark.parametrize("over", [
    dict(O=0), dict(O=2 ** 24 + 1, os=2 ** 25), dict(H=0), dict(H=131057, ws=131072, xs=131072),
    dict(ws=56), dict(ws=32), dict(ws=2 ** 22 + 16), dict(w=None), dict(w=0x10008),
    dict(scale=None), dict(type=0), dict(type=4), dict(out_type=3), dict(out_type=-1), dict(T=-1),
    dict(T=2 ** 24 + 1), dict(x=None), dict(xs=39), dict(out=None), dict(os=23), dict(work=None),
    dict(work=0x50008), dict(out=0x30000 + 318),
    dict(Q, xs=40), dict(Q, xs=56), dict(Q, xs=2 ** 22 + 16), dict(Q, x=0x30008),
    dict(Q, x_scales=None), dict(Q, out=0x60000), dict(Q, out=0x30000 + 190)], ids=str)
def test_linear8_rejects(lib, over):
    assert _linear(lib, **over) == -1


def _moe8(lib, **over):
    f = dict(S=4, H=32, I=16, type=1, weights=3, w13=0x10000, w2=0x20000, s13=0x21000, s2=0x22000)
    f.update({k: v for k, v in over.items() if k in f})
    e = _lib.Experts(*f.values())
    a = dict(x=0x30000, xs=32, probs=0x40000, ids=0x50000, id_bytes=4, T=2, k=2, out=0x60000,
             os=32, work=0x70000)
    a.update({k: v for k, v in over.items() if k in a})
    if "bytes" in over:
        size = ctypes.c_long(-5)
        return lib.expert_cache_moe8_workspace(ctypes.addressof(e), a["T"], a["k"],
                                               ctypes.addressof(size))
    return lib.expert_cache_moe8(ctypes.addressof(e), *a.values(), None)


BAD_LAYER = [dict(S=0), dict(S=1025), dict(H=0), dict(I=0), dict(H=40), dict(I=24), dict(H=131072),
             dict(I=131072), dict(type=0), dict(type=3), dict(weights=1), dict(weights=4),
             dict(H=65536, I=16384), dict(T=-1), dict(k=0), dict(k=65), dict(T=2 ** 24, k=2),
             dict(T=2 ** 23, H=1024)]


@pytest.mark.parametrize("over", BAD_LAYER + [
    dict(w13=None), dict(w2=None), dict(w13=0x10008), dict(w2=0x20004), dict(s13=None),
    dict(s2=None), dict(x=None), dict(xs=31), dict(out=None), dict(os=31), dict(probs=None),
    dict(ids=None), dict(id_bytes=2), dict(work=None), dict(work=0x70008), dict(out=0x30000 + 126),
    dict(out=0x40000), dict(out=0x50000)], ids=str)
def test_moe8_rejects(lib, over):
    assert _moe8(lib, **over) == -1


@pytest.mark.parametrize("over", BAD_LAYER, ids=str)
def test_moe8_workspace_rejects(lib, over):
    assert _moe8(lib, bytes=True, **over) == -1


# A launch has less than 2^32 threads: what would need more is refused before the first of a call.
@pytest.mark.parametrize("entry,over", [
    (_dispatch, dict(T=2 ** 24, k=1, H=1025, xs=1025, os=1025)),
    (_dispatch, dict(T=2 ** 23, k=1, type=0, H=1025, xs=1025, os=1025)),
    (_combine, dict(T=2 ** 24, k=1, H=1025, ys=1025, os=1025)),
    (_combine_grad, dict(T=2 ** 24, k=1, H=1025, gs=1025, ys=1025, ds=1025)),
    (_quantize, dict(T=2 ** 23 + 1)), (_linear, dict(T=2 ** 23 + 1)),
    (_linear, dict(T=2 ** 23, O=2 ** 15 + 1, os=2 ** 16)), (_moe8, dict(T=2 ** 23 + 1, k=1)),
    (_moe8, dict(T=2 ** 20 + 1, k=64, I=1024)), (_moe8, dict(T=2 ** 22, k=2, I=8208)),
    (_moe8, dict(T=2 ** 17, k=64, H=8208, xs=8208, os=8208)),
    (_moe8, dict(bytes=True, T=2 ** 22, k=2, I=8208)),
    (_moe8, dict(bytes=True, T=2 ** 23 + 1, k=1))], ids=str)
def test_calls_of_more_than_a_launch_holds_are_rejected(lib, entry, over):
    assert entry(lib, **over) == -1


def test_null_handles_are_rejected(lib):
    size = ctypes.c_long()
    at = ctypes.addressof(size)
    assert lib.expert_cache_linear8_workspace(None, 1, 1, at) == -1
    assert lib.expert_cache_moe8_workspace(None, 1, 1, at) == -1
    assert lib.expert_cache_linear8(None, 16, 1, 32, None, 1, 16, 1, 32, 16, None) == -1
    assert lib.expert_cache_moe8(None, 16, 32, 16, 16, 4, 1, 1, 16, 32, 16, None) == -1
    l = _lib.Linear(24, 40, 48, 16, 16, None)
    assert lib.expert_cache_linear8_workspace(ctypes.addressof(l), 1, 1, None) == -1


def test_nothing_to_do_is_no_call(lib):
    assert _dispatch(lib, T=0, x=None, out=None, places=None, rows=None) == 0
    assert _combine(lib, T=0, y=None, out=None, places=None) == 0
    assert _combine_grad(lib, T=0, g=None, y=None, places=None, rows=None) == 0
    assert _quantize(lib, T=0, x=None, q=None, scales=None) == 0
    assert _linear(lib, T=0, x=None, out=None, work=None) == 0
    assert _moe8(lib, T=0, x=None, out=None, ids=None, work=None) == 0


def test_workspaces_cover_what_is_written(lib):
    size = ctypes.c_long()
    at = ctypes.addressof(size)
    for T, O, H in ((1, 1, 1), (77, 24, 1045), (2 ** 20, 8, 131056)):
        l = _lib.Linear(O, H, -(-H // 16) * 16, 16, 16, None)
        assert lib.expert_cache_linear8_workspace(ctypes.addressof(l), 1, T, at) == 0
        assert size.value >= T * -(-H // 16) * 16 + 4 * T
        assert lib.expert_cache_linear8_workspace(ctypes.addressof(l), 3, T, at) == 0
    for T, k, S, H, I in ((1, 1, 1, 16, 16), (2048, 8, 128, 2048, 768), (2 ** 20, 2, 8, 1024, 4096)):
        e = _lib.Experts(S, H, I, 1, 3, 16, 16, 16, 16)
        assert lib.expert_cache_moe8_workspace(ctypes.addressof(e), T, k, at) == 0
        # tokens and hidden values in 8 bits, hidden values and outputs in 32, places and rows
        assert size.value >= T * H + T * k * (I + 4 * max(H, I) + 8)


# ---- Python -------------------------------------------------------------------------------

@pytest.fixture
def anywhere(monkeypatch):
    """Lets CPU tensors past the device check, so that the checks after it are reached."""
    monkeypatch.setattr(ops, "_on_gpu", lambda *t: t[0].device)


def _order(T=3, k=2, S=4):
    return ops.Order(torch.zeros(S + 1, dtype=torch.int32), torch.zeros(T * k, dtype=torch.int32),
                     torch.zeros((T, k), dtype=torch.int32), S)


@pytest.fixture
def order(anywhere):
    return _order()


@pytest.mark.parametrize("offsets,rows,places,S", [
    (5, 6, (3, 2), 3), (5, 5, (3, 2), 4), (5, 6, (6,), 4), (5, 0, (3, 0), 4), (1, 6, (3, 2), 0),
    (1026, 6, (3, 2), 1025), (5, 195, (3, 65), 4)], ids=range(7))
def test_orders(anywhere, offsets, rows, places, S):
    t = [torch.zeros(n, dtype=torch.int32) for n in (offsets, rows, places)]
    with pytest.raises(ValueError):
        ops.Order(*t, S)


def test_orders_of_other_types(anywhere):
    for i in range(3):
        t = [torch.zeros(n, dtype=torch.int32) for n in (5, 6, (3, 2))]
        ops.Order(*t, 4)
        t[i] = t[i].long()
        with pytest.raises(ValueError):
            ops.Order(*t, 4)
    with pytest.raises(ValueError):
        ops.Order(torch.zeros(10, dtype=torch.int32)[::2], *t[1:2],
                  torch.zeros((3, 2), dtype=torch.int32), 4)


def test_tensors_on_the_host_are_refused():
    for call in (lambda: ops.sort(torch.zeros((2, 2), dtype=torch.int32), 2),
                 lambda: ops.quantize(torch.zeros(2, 8, dtype=BF16)),
                 lambda: ops.Linear8(torch.zeros(2, 16, dtype=I8), torch.ones(2)),
                 lambda: ops.Experts8(*_w(), *_s()), _order):
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.mark.parametrize("ids,S", [
    (torch.zeros(2, 2, 2, dtype=torch.int32), 2), (torch.tensor(1), 2),
    (torch.zeros(2, 65, dtype=torch.int32), 2), (torch.zeros(2, 0, dtype=torch.int32), 2),
    (torch.zeros(2, 2, dtype=torch.int32), 0), (torch.zeros(2, 2, dtype=torch.int32), 1025),
    (torch.zeros(2, 2, dtype=torch.int16), 2), (torch.zeros(2, 2), 2),
    (torch.zeros(1, 1, dtype=torch.int32).expand(2 ** 24, 2), 2)], ids=range(9))
def test_sort_arguments(anywhere, ids, S):
    with pytest.raises(ValueError):
        ops.sort(ids, S)


@pytest.mark.parametrize("x", [
    torch.zeros(4, 8), torch.zeros(3, 8, dtype=torch.float64), torch.zeros(3, 8, dtype=torch.int32),
    torch.zeros(24), torch.zeros(3, 0), torch.zeros(1, 1).expand(3, 2 ** 20 + 1),
    torch.zeros(3, 8, device="meta")], ids=range(7))
def test_dispatch_arguments(order, x):
    for wants in (False, True):
        x = x.detach().requires_grad_(wants and x.is_floating_point())
        with pytest.raises(ValueError):
            ops.dispatch(x, order)


def test_more_rows_than_a_launch_moves_are_refused(anywhere):
    order = ops.Order(torch.zeros(5, dtype=torch.int32), torch.zeros(2 ** 20, dtype=torch.int32),
                      torch.zeros((2 ** 20, 1), dtype=torch.int32), 4)
    for dtype, H in ((BF16, 16385), (F32, 8193)):
        rows = torch.zeros(1, 1, dtype=dtype).expand(2 ** 20, H)
        for call in (lambda: ops.dispatch(rows, order), lambda: ops.combine(rows, None, order),
                     lambda: ops.combine_grad(rows, rows, None, order)):
            with pytest.raises(ValueError, match="bytes"):
                call()


def test_more_tokens_than_a_launch_holds_are_refused(anywhere):
    one = torch.zeros(1, 1, dtype=BF16)
    with pytest.raises(ValueError, match="rows"):
        ops.quantize(one.expand(2 ** 23 + 1, 1))
    with pytest.raises(ValueError, match="tokens"):
        _lin()(one.expand(2 ** 23 + 1, 32))
    layer = ops.Experts8(*_w(I=1024), *_s(I=1024))
    for T, k, of in ((2 ** 23 + 1, 1, layer), (2 ** 20, 64, layer),
                     (2 ** 22, 2, ops.Experts8(*_w(I=8208), *_s(I=8208)))):
        with pytest.raises(ValueError, match="pairs"):
            of(one.expand(T, 32), torch.zeros(1, 1).expand(T, k),
               torch.zeros(1, 1, dtype=torch.int32).expand(T, k))


@pytest.mark.parametrize("y,w", [
    (torch.zeros(5, 8), None), (torch.zeros(6, 8, dtype=torch.float64), None),
    (torch.zeros(6, 8), torch.zeros(3, 2, dtype=BF16)), (torch.zeros(6, 8), torch.zeros(2, 3)),
    (torch.zeros(6, 8), torch.zeros(6)), (torch.zeros(6, 8), torch.zeros(3, 2, device="meta"))],
    ids=range(6))
def test_combine_arguments(order, y, w):
    for wants in (False, True):
        with pytest.raises(ValueError):
            ops.combine(y.detach().requires_grad_(wants), w, order)
    with pytest.raises(ValueError):
        ops.combine_grad(torch.zeros(3, 8), y, w, order)


def test_combine_grad_arguments(order):
    g, y, w = torch.zeros(3, 8), torch.zeros(6, 8), torch.zeros(3, 2)
    for bad in ((torch.zeros(4, 8), y, w), (g.to(BF16), y, w), (g, torch.zeros(6, 9), w),
                (g, None, w), (g.double(), y, w)):
        with pytest.raises(ValueError):
            ops.combine_grad(*bad, order)
    with pytest.raises(ValueError, match="weights"):
        ops.combine_grad(g, None, torch.zeros(2, 3), _order(), need_weights=False)
    assert ops.combine_grad(g, y, None, _order(), need_y=False) == (None, None)
    for i in range(3):
        t = [g.clone(), y.clone(), w.clone()]
        t[i].requires_grad_()
        with pytest.raises(ValueError, match="backward"):
            ops.combine_grad(*t, order)


def test_recording_is_refused_while_a_graph_is_captured(order, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    x, y = torch.zeros(3, 8, requires_grad=True), torch.zeros(6, 8, requires_grad=True)
    w = torch.zeros(3, 2, requires_grad=True)
    for call in (lambda: ops.dispatch(x, order), lambda: ops.combine(y, None, order),
                 lambda: ops.combine(y.detach(), w, order)):
        with pytest.raises(ValueError, match="captured"):
            call()


@pytest.mark.parametrize("x", [
    torch.zeros(2, 8), torch.zeros(8, dtype=BF16), torch.zeros(2, 0, dtype=BF16),
    torch.zeros(1, 1, dtype=BF16).expand(1, 2 ** 20 + 1),
    torch.zeros(1, 1, dtype=BF16).expand(2 ** 24 + 1, 1)], ids=range(5))
def test_quantize_arguments(anywhere, x):
    with pytest.raises(ValueError):
        ops.quantize(x)


def _lin(O=6, H=32, **kw):
    return ops.Linear8(torch.zeros(O, H, dtype=I8), torch.ones(O), **kw)


@pytest.mark.parametrize("make", [
    lambda: ops.Linear8(torch.zeros(6, 32), torch.ones(6)),
    lambda: ops.Linear8(torch.zeros(6, dtype=I8), torch.ones(6)),
    lambda: ops.Linear8(torch.zeros(0, 32, dtype=I8), torch.ones(0)),
    lambda: ops.Linear8(torch.zeros(6, 32, dtype=I8), torch.ones(5)),
    lambda: ops.Linear8(torch.zeros(6, 32, dtype=I8), torch.ones(6, dtype=BF16)),
    lambda: ops.Linear8(torch.zeros(6, 32, dtype=I8), torch.ones(12)[::2]),
    lambda: ops.Linear8(torch.zeros(1, 131057, dtype=I8), torch.ones(1)),
    lambda: _lin(bias=torch.ones(5)), lambda: _lin(bias=torch.ones(6, 1)),
    lambda: _lin(bias=torch.ones(6, dtype=torch.float64)),
], ids=range(10))
def test_linear8_weights(anywhere, make):
    with pytest.raises(ValueError):
        make()


X8 = dict(x=torch.zeros(3, 32, dtype=I8), x_scales=torch.ones(3))


@pytest.mark.parametrize("kw", [
    dict(x=torch.zeros(3, 31, dtype=BF16)), dict(x=torch.zeros(32, dtype=BF16)),
    dict(x=torch.zeros(3, 32)), dict(x=torch.zeros(3, 32, dtype=BF16, device="meta")),
    dict(x=torch.zeros(3, 32, dtype=BF16), x_scales=torch.ones(3)), dict(X8, x_scales=None),
    dict(X8, x_scales=torch.ones(4)), dict(X8, x_scales=torch.ones(3, dtype=BF16)),
    dict(X8, x_scales=torch.ones(3, 1)), dict(X8, dtype=torch.float64), dict(X8, dtype=I8),
    dict(X8, out=torch.zeros(3, 6)), dict(X8, dtype=F16, out=torch.zeros(2, 6, dtype=F16)),
    dict(X8, out=torch.zeros(6, 3, dtype=BF16).t())], ids=range(14))
def test_linear8_arguments(anywhere, kw):
    with pytest.raises(ValueError):
        _lin()(**kw)


def test_linear8_takes_weights_as_they_lie_or_lays_them_out(anywhere):
    w = torch.arange(6 * 64).view(6, 64).to(I8)
    scale = torch.ones(6, 1)
    for of in (w, w[:, :32], w[:, 16:48], w[::2]):
        lin = ops.Linear8(of, scale[:of.shape[0]])
        if of.data_ptr() % 16 == 0:
            assert lin.w.data_ptr() == of.data_ptr()
    for of in (w[:, :33], w[:, 1:33], w.t()[:6, :6], w[:, ::2]):
        lin = ops.Linear8(of, scale)
        assert lin.w.data_ptr() != of.data_ptr() and lin.w.shape[1] % 16 == 0
        assert torch.equal(lin.w[:, :of.shape[1]], of) and not lin.w[:, of.shape[1]:].any()
        assert lin.H == of.shape[1]


def _w(S=2, H=32, I=16, dtype=I8):
    return torch.zeros(S, 2 * I, H).to(dtype), torch.zeros(S, H, I).to(dtype)


def _s(S=2, H=32, I=16):
    return torch.ones(S, 2 * I), torch.ones(S, H)


@pytest.mark.parametrize("make", [
    lambda: ops.Experts8(_w()[0][0], _w()[1], *_s()), lambda: ops.Experts8(*_w(dtype=BF16), *_s()),
    lambda: ops.Experts8(_w()[0][:, :31], _w()[1], *_s()),
    lambda: ops.Experts8(_w()[0], _w(S=3)[1], *_s()),
    lambda: ops.Experts8(*_w(H=40), *_s(H=40)), lambda: ops.Experts8(*_w(I=24), *_s(I=24)),
    lambda: ops.Experts8(*_w(S=1025, H=16), *_s(S=1025, H=16)),
    lambda: ops.Experts8(*_w(), _s()[0], None), lambda: ops.Experts8(*_w(), *_s(S=3)),
    lambda: ops.Experts8(*_w(), _s()[0].to(BF16), _s()[1]),
    lambda: ops.Experts8(torch.zeros(2, 32, 33, dtype=I8)[:, :, :32], _w()[1], *_s()),
    lambda: ops.Experts8(torch.empty(1, 32, 131072, dtype=I8),
                         torch.empty(1, 131072, 16, dtype=I8), *_s(1, 131072)),
], ids=range(12))
def test_experts8_weights(anywhere, make):
    with pytest.raises(ValueError):
        make()


def _call(T=3, k=2, H=32, dtype=BF16, ids=torch.int32):
    return [torch.zeros(T, H, dtype=dtype), torch.zeros(T, k), torch.zeros(T, k, dtype=ids)]


@pytest.mark.parametrize("x,p,i,out", [
    (*_call(H=16), None), (*_call(dtype=F32), None), (*_call(ids=torch.int16), None),
    (*_call(T=1, k=65), None), (*_call(k=0), None), (_call()[0], _call(k=3)[1], _call()[2], None),
    (_call()[0], _call(T=2)[1], _call(T=2)[2], None),
    (_call()[0], _call()[1].to(BF16), _call()[2], None),
    (_call()[0], *[t[0] for t in _call()[1:]], None),
    (*_call(), torch.zeros(3, 32, dtype=F16)), (*_call(), torch.zeros(2, 32, dtype=BF16)),
    (*_call(), torch.zeros(32, 3, dtype=BF16).t()),
    (torch.zeros(1, 1, dtype=BF16).expand(2 ** 26, 32), torch.zeros(1, 1).expand(2 ** 26, 1),
     torch.zeros(1, 1, dtype=torch.int32).expand(2 ** 26, 1), None),
], ids=range(13))
def test_experts8_arguments(anywhere, x, p, i, out):
    with pytest.raises(ValueError):
        ops.Experts8(*_w(), *_s())(x, p, i, out)


@pytest.fixture
def no_kernels(anywhere, monkeypatch):
    """Calls that every check lets through, without a device."""
    calls = []
    monkeypatch.setattr(ops, "_on_device", lambda device, call, *args: calls.append(args) or 0)
    return calls


GRAD_CALLS = {
    "quantize": (lambda t: ops.quantize(t["x"]), ("x",)),
    "linear8": (lambda t: ops.Linear8(t["w"], t["s"], t["b"])(t["x"], out=t["out"]),
                ("s", "b", "x", "out")),
    "whole": (lambda t: ops.Linear8(t["w"], t["s"])(t["q"], t["qs"]), ("s", "qs")),
    "experts8": (lambda t: ops.Experts8(t["w13"], t["w2"], t["s13"], t["s2"])(t["x"], t["p"], t["i"]),
                 ("s13", "s2", "x", "p")),
}


@pytest.mark.parametrize("op,name", [(op, n) for op, (_, names) in GRAD_CALLS.items()
                                     for n in names])
def test_what_needs_a_gradient_is_refused(no_kernels, op, name):
    x, p, i = _call()
    w13, w2 = _w()
    s13, s2 = _s()
    t = dict(x=x, p=p, i=i, w13=w13, w2=w2, s13=s13, s2=s2, w=torch.zeros(6, 32, dtype=I8),
             s=torch.ones(6), b=torch.ones(6), out=torch.zeros(3, 6, dtype=BF16),
             q=torch.zeros(3, 32, dtype=I8), qs=torch.ones(3))
    call = GRAD_CALLS[op][0]
    call(t)
    t[name].requires_grad_()
    with pytest.raises(ValueError, match="backward"):
        call(t)
    assert len(no_kernels) == 1
    with torch.no_grad():
        call(t)
    t[name] = t[name].detach()
    call(t)
    assert len(no_kernels) == 3

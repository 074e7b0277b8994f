"""Calls at the edges of what the operators for many tokens take (vllm_expert_cache/ops.py and their C
entry points), checked without a GPU: none of them launches a kernel."""
from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from vllm_expert_cache import _lib, ops

BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


@pytest.fixture
def no_kernels(monkeypatch):
    """Lets CPU tensors past the device check, and calls that every check lets through end without
    a device."""
    calls = []
    monkeypatch.setattr(ops, "_on_gpu", lambda *t: t[0].device)
    monkeypatch.setattr(ops, "_on_device", lambda device, call, *args: calls.append(args) or 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return calls


# ---- no tokens ----------------------------------------------------------------------------

# few and many outputs, of lengths that are cut where tokens are few (6017 on) and that aren't
@pytest.mark.parametrize("H", [16, 6000, 6017, 131056])
@pytest.mark.parametrize("O", [1, 8191, 8192, 2 ** 24])
def test_a_projection_of_no_tokens(lib, no_kernels, O, H):
    size = ctypes.c_long(-5)
    l = _lib.Linear(O, H, -(-H // 16) * 16, 16, 16, None)
    for kind in (1, 2, 3):
        size.value = -5
        assert lib.expert_cache_linear8_workspace(ctypes.addressof(l), kind, 0,
                                                  ctypes.addressof(size)) == 0
        assert size.value == 0
    if O == 8192 and H < 10000:
        lin = ops.Linear8(torch.zeros((O, H), dtype=I8), torch.ones(O))
        assert lin(torch.empty((0, H), dtype=BF16)).shape == (0, O)
        assert lin(torch.empty((0, H), dtype=I8), torch.empty(0)).shape == (0, O)


def test_a_layer_of_no_tokens(lib):
    size = ctypes.c_long(-5)
    for S, H, I in ((1, 16, 16), (1024, 131056, 16)):
        e = _lib.Experts(S, H, I, 1, 3, 16, 16, 16, 16)
        assert lib.expert_cache_moe8_workspace(ctypes.addressof(e), 0, 8, ctypes.addressof(size)) == 0


# ---- forward-mode derivatives -------------------------------------------------------------

def _order(T=3, k=2, S=4):
    return ops.Order(torch.zeros(S + 1, dtype=torch.int32), torch.zeros(T * k, dtype=torch.int32),
                     torch.zeros((T, k), dtype=torch.int32), S)


def _tensors():
    """Arguments of every operator; those that may be floating point can have a tangent."""
    return dict(
        x=torch.zeros(3, 32, dtype=BF16), y=torch.zeros(6, 32, dtype=BF16),
        g=torch.zeros(3, 32, dtype=BF16), p=torch.zeros(3, 2),
        i=torch.zeros(3, 2, dtype=torch.int32), i1=torch.zeros(3, dtype=torch.int32),
        logits=torch.zeros(3, 16), gate=torch.zeros(16), w=torch.zeros(6, 32, dtype=I8),
        s=torch.ones(6), b=torch.ones(6), b16=torch.ones(6, dtype=BF16),
        q=torch.zeros(3, 32, dtype=I8), qs=torch.ones(3), out6=torch.zeros(3, 6, dtype=BF16),
        out32=torch.zeros(3, 32, dtype=BF16), base=torch.zeros(3, 6, dtype=BF16),
        w13=torch.zeros(2, 32, 32, dtype=I8), w2=torch.zeros(2, 32, 16, dtype=I8),
        s13=torch.ones(2, 32), s2=torch.ones(2, 32), v13=torch.zeros(2, 32, 32, dtype=BF16),
        v2=torch.zeros(2, 32, 16, dtype=BF16), down=torch.zeros(2, 8, 32, dtype=BF16),
        up=torch.zeros(2, 6, 8, dtype=BF16), factors=torch.ones(2))


# (call, the arguments that can have a tangent)
CALLS = {
    "route": (lambda t: ops.route(t["logits"], 2, bias=t["gate"]), ("logits", "gate")),
    "dispatch": (lambda t: ops.dispatch(t["x"], _order()), ("x",)),
    "combine": (lambda t: ops.combine(t["y"], t["p"], _order()), ("y", "p")),
    "combine_grad": (lambda t: ops.combine_grad(t["g"], t["y"], t["p"], _order()), ("g", "y", "p")),
    "quantize": (lambda t: ops.quantize(t["x"]), ("x",)),
    "linear8": (lambda t: ops.Linear8(t["w"], t["s"], t["b"])(t["x"], out=t["out6"]),
                ("x", "s", "b", "out6")),
    "linear8 copied": (lambda t: ops.Linear8(t["w"], t["s"], t["b16"])(t["x"]), ("b16",)),
    "linear8 whole": (lambda t: ops.Linear8(t["w"], t["s"])(t["q"], t["qs"]), ("qs", "s")),
    "experts8": (lambda t: ops.Experts8(t["w13"], t["w2"], t["s13"], t["s2"])(
        t["x"], t["p"], t["i"], out=t["out32"]), ("x", "p", "s13", "s2", "out32")),
    "experts": (lambda t: ops.Experts(t["v13"], t["v2"])(t["x"], t["p"], t["i"], out=t["out32"]),
                ("x", "p", "v13", "v2", "out32")),
    "experts int8": (lambda t: ops.Experts(t["w13"], t["w2"], t["s13"], t["s2"])(
        t["x"], t["p"], t["i"]), ("x", "s13", "s2")),
    "adapters": (lambda t: ops.Adapters(t["down"], t["up"], t["factors"])(
        t["x"], t["base"], t["i1"], out=t["out6"]),
        ("x", "base", "down", "up", "factors", "out6")),
}
TANGENTS = [(op, name) for op, (_, names) in CALLS.items() for name in names]


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("op,name", TANGENTS)
def test_a_tangent_is_refused_and_not_dropped(no_kernels, op, name, no_grad):
    call, t = CALLS[op][0], _tensors()
    with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
        call(t)  # a level alone changes nothing
        assert len(no_kernels) == 1
        primal = t[name]
        t[name] = forward_ad.make_dual(primal, torch.ones_like(primal))
        with pytest.raises(ValueError, match="forward-mode"):
            call(t)
        assert len(no_kernels) == 1
        t[name] = forward_ad.unpack_dual(t[name]).primal
        call(t)
    assert len(no_kernels) == 2


@pytest.mark.parametrize("of", ["dispatch", "combine"])
def test_a_tangent_of_a_gradient_is_refused(no_kernels, of):
    """Forward over reverse: the backward pass is a call like any other."""
    leaf = torch.zeros((3, 32) if of == "dispatch" else (6, 32), requires_grad=True)
    weights = torch.zeros(3, 2, requires_grad=True)
    out = ops.dispatch(leaf, _order()) if of == "dispatch" else ops.combine(leaf, weights, _order())
    with forward_ad.dual_level():
        grad = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(ValueError, match="forward-mode"):
            torch.autograd.grad(out, leaf, grad, retain_graph=True)
        assert len(no_kernels) == 1
        torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert len(no_kernels) == 2


# ---- traces -------------------------------------------------------------------------------

TRACED = {name: call for name, (call, _) in CALLS.items()}
TRACED["sort"] = lambda t: ops.sort(t["i"], 4)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
@pytest.mark.parametrize("op", TRACED)
@pytest.mark.parametrize("how", ["trace", "make_fx"])
def test_a_trace_is_refused(monkeypatch, op, how):
    """It would hold the allocation of the result and nothing that fills it."""
    from torch.fx.experimental.proxy_tensor import make_fx

    class Library:
        launches = []

        def __getattr__(self, name):
            if name.endswith("_workspace"):
                return lambda *args: 0
            return lambda *args: self.launches.append(name) or 0

    library, t = Library(), _tensors()
    monkeypatch.setattr(ops._lib, "lib", lambda: library)
    monkeypatch.setattr(ops, "_on_gpu", lambda *t: t[0].device)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: None)
    monkeypatch.setattr(ops, "_workspace", lambda *args: 16)

    def of(x):
        out = TRACED[op](t)
        return out.places if op == "sort" else out[0] if isinstance(out, tuple) else out

    of(t["x"])
    assert len(library.launches) == 1
    with pytest.raises(ValueError, match="trace"):
        if how == "trace":
            torch.jit.trace(of, t["x"], check_trace=False)
        else:
            make_fx(of)(t["x"])
    assert len(library.launches) == 1
    of(t["x"])
    assert len(library.launches) == 2


# ---- results that meet what the call reads ------------------------------------------------

S, H, I, T, K = 4, 32, 16, 2, 2
LAYER = dict(w13=(0x10000, S * 2 * I * H), w2=(0x20000, S * H * I), s13=(0x30000, 4 * S * 2 * I),
             s2=(0x40000, 4 * S * H), x=(0x50000, 2 * T * H), probs=(0x60000, 4 * T * K),
             ids=(0x70000, 4 * T * K), work=(0x80000, None))


def _workspace_of(lib):
    size = ctypes.c_long()
    e = _lib.Experts(S, H, I, 1, 3, 16, 16, 16, 16)
    assert lib.expert_cache_moe8_workspace(ctypes.addressof(e), T, K, ctypes.addressof(size)) == 0
    return size.value


@pytest.mark.parametrize("name", LAYER)
def test_a_layers_result_over_what_it_reads_is_refused(lib, name):
    """Its first byte on the array's last, and its last on the array's first: -1, before any launch."""
    at = {n: first for n, (first, _) in LAYER.items()}
    first, size = LAYER[name]
    size = _workspace_of(lib) if size is None else size
    e = _lib.Experts(S, H, I, 1, 3, at["w13"], at["w2"], at["s13"], at["s2"])
    for out in (first + size - 1, first - 2 * T * H + 1):
        assert lib.expert_cache_moe8(ctypes.addressof(e), at["x"], H, at["probs"], at["ids"], 4, T, K,
                                     out, H, at["work"], None) == -1


# ---- a caller's `out` ---------------------------------------------------------------------

INTO = {"linear8": "out6", "experts8": "out32", "experts": "out32", "adapters": "out6"}


@pytest.mark.parametrize("op", INTO)
def test_a_write_into_out_is_counted(no_kernels, op):
    """A backward pass that saved `out` before finds that it was written since."""
    t = _tensors()
    out, factor = t[INTO[op]], torch.ones((), dtype=BF16, requires_grad=True)
    product = out * factor
    CALLS[op][0](t)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with torch.inference_mode():  # where nothing is counted
        t[INTO[op]] = torch.empty_like(out)
        CALLS[op][0](t)
    assert len(no_kernels) == 2


# ---- workspaces ---------------------------------------------------------------------------

# tokens, outputs, length and parts of it: as many as have room beside each other (256 tiles of 64 x
# 64), as leave each eight steps of 128, and eight at most
@pytest.mark.parametrize("T,O,H,parts", [(70, 130, 6200, 6), (130, 1029, 6160, 5), (20, 77, 8300, 8),
                                         (64, 4096, 14336, 4), (1, 8192, 6017, 2), (1, 8192, 6016, 1),
                                         (1, 8193, 8192, 1), (1, 10, 131056, 1)])
def test_workspaces_hold_the_parts_of_a_length(lib, T, O, H, parts):
    K = -(-H // 16) * 16
    l, size = _lib.Linear(O, H, K, 16, 16, None), ctypes.c_long()
    sums = 4 * parts * T * -(-O // 4) * 4 if parts > 1 else 0
    assert lib.expert_cache_linear8_workspace(ctypes.addressof(l), 3, T, ctypes.addressof(size)) == 0
    assert size.value == sums
    assert lib.expert_cache_linear8_workspace(ctypes.addressof(l), 1, T, ctypes.addressof(size)) == 0
    assert size.value >= T * K + 4 * T + sums

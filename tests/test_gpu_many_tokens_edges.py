"""The operators for many tokens (vllm_expert_cache/ops.py) on the GPU where their plans change: one row
through parts of a length, long products in every tile, slots that just fill a small tile, many
tiles. Against the formulas in 64 bits and the tolerances of `test_gpu_many_tokens.py`."""
from __future__ import annotations

import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import gpu_util as gu
import test_gpu_many_tokens as many
from vllm_expert_cache import _lib, ops

pytestmark = pytest.mark.gpu

DEV = gu.DEV
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def _workspace(lin, kind, T):
    size = ctypes.c_long()
    assert _lib.lib().expert_cache_linear8_workspace(lin._at, kind, T, ctypes.addressof(size)) == 0
    return size.value


# ---- linear8 ------------------------------------------------------------------------------

def test_a_projection_of_no_tokens():
    """As long, and of as many outputs, as is cut along the length where there are tokens."""
    lin = ops.Linear8(torch.ones((8192, 6208), dtype=I8, device=DEV), torch.ones(8192, device=DEV))
    assert lin(torch.empty((0, 6208), dtype=BF16, device=DEV)).shape == (0, 8192)
    assert lin(torch.empty((0, 6208), dtype=I8, device=DEV),
               torch.empty(0, device=DEV)).shape == (0, 8192)


# 49, 48 and 64 steps in two parts: 8192 outputs are 128 tiles, so two of each are beside each other
@pytest.mark.parametrize("H", [6211, 6017, 8192])
@pytest.mark.parametrize("dtype", [BF16, I8])
def test_one_row_of_any_stride_in_parts_of_its_length(H, dtype):
    g, O = many._gen(H), 8192
    w = many._whole(g, O, H)
    lin = ops.Linear8(w, torch.rand(O, device=DEV, generator=g), many._randn(g, O))
    x, s = many._randn(g, 1, H).to(BF16), None
    want, bound = many._linear(*many._quantized(x), lin, lin.bias)
    if dtype == I8:
        x, s = ops.quantize(x)
    kind, size = (1, _workspace(lin, 1, 1)) if dtype == BF16 else (3, _workspace(lin, 3, 1))
    assert size >= 4 * 2 * O  # both parts' sums
    work = torch.empty(size, dtype=torch.uint8, device=DEV)
    for x_stride, out_stride in ((0, 0), (16, 4), (x.stride(0), O), (2 ** 22, 2 ** 20)):
        out = torch.full((O + 64,), 7.0, device=DEV)
        torch.cuda.synchronize()
        assert _lib.lib().expert_cache_linear8(
            lin._at, x.data_ptr(), kind, x_stride, None if s is None else s.data_ptr(), 1,
            out.data_ptr(), 0, out_stride, work.data_ptr(), None) == 0
        torch.cuda.synchronize()
        many._close(out[None, :O], want, bound + many.HALF[F32] * (want.abs() + bound))
        assert (out[O:] == 7).all()


# tiles of 128 and of 256, of 9 steps with a tail, 9 whole ones and a chunk, and 17: every stage
# loaded again and again
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,H,O", [(1000, 1045, 2344), (1100, 1152, 2043), (2500, 1040, 2568),
                                   (2437, 1045, 2701), (2304, 2064, 2816)])
def test_long_products_in_large_tiles(T, H, O, dtype):
    g = many._gen(T + H + O)
    bias = many._randn(g, O) if O % 2 else None
    w = many._whole(g, O, H)
    lin = ops.Linear8(w, (0.5 + torch.rand(O, device=DEV, generator=g)) * H ** -0.5 / 40, bias)
    x = many._randn(g, T, H).to(dtype)
    want, bound = many._linear(*many._quantized(x), lin, bias)
    for out in (dtype, F32):
        y = lin(x, dtype=out)
        many._close(y, want, bound + many.HALF[out] * (want.abs() + bound) + many.TINY[out])
    assert torch.equal(lin(x), lin(x))


@pytest.mark.parametrize("T,H,O", [(1, 6017, 8192), (130, 6160, 1029), (1000, 1045, 2344),
                                   (2437, 272, 2701)])
def test_a_projection_captured(T, H, O):
    """Parts with their join, and both large tiles: every replay gives the eager call's bits."""
    g = many._gen(T)
    lin = ops.Linear8(many._whole(g, O, H), torch.rand(O, device=DEV, generator=g))
    x = many._randn(g, T, H).to(BF16)
    lin(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lin(x)
    for _ in range(4):
        x.copy_(many._randn(g, T, H))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, lin(x))


# ---- experts8 -----------------------------------------------------------------------------

def test_experts8_of_every_fill_of_small_tiles():
    """Slots of as many pairs as fill tiles of 64 rows, their rounds and their operands, and one
    more or less, between slots of none."""
    fills = many.FILLS + [0] * 20
    S, H, I = len(fills), 144, 80
    assert sum(fills) <= 96 * S  # which is what makes tiles of 64 rows
    e = many._experts(90, S, H, I)
    g = many._gen(91)
    ids = torch.repeat_interleave(torch.randperm(S, device=DEV, generator=g),
                                  torch.tensor(fills, device=DEV))
    ids = ids[torch.randperm(len(ids), device=DEV, generator=g)].unsqueeze(1)
    x = many._randn(g, len(ids), H).to(BF16)
    probs = torch.rand((len(ids), 1), device=DEV, generator=g) + 0.1
    got = e(x, probs, ids)
    many._close(got, *many._moe8(e, x, probs, ids))
    assert torch.equal(got, e(x, probs, ids))


def test_experts8_of_many_tiles_of_256_rows():
    T, k, S, H, I = 33000, 2, 8, 1024, 48
    assert T * k >= 256 * S
    e = many._experts(92, S, H, I)
    x, probs, ids = many._tokens(93, T, k, S, H, BF16, torch.int32)
    got = e(x, probs, ids)
    many._close(got, *many._moe8(e, x, probs, ids))
    some = torch.arange(0, T, 997, device=DEV)
    assert torch.equal(e(x[some], probs[some], ids[some]), got[some])


# ---- autograd -----------------------------------------------------------------------------

@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
def test_tangents_and_traces_are_refused():
    order = ops.sort(many._ids(many._gen(94), 5, 2, 3), 3)
    x = torch.ones((5, 8), device=DEV)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(ValueError, match="forward-mode"):
            ops.dispatch(dual, order)
        assert torch.equal(ops.dispatch(forward_ad.unpack_dual(dual).primal, order),
                           ops.dispatch(x, order))
    with pytest.raises(ValueError, match="trace"):
        torch.jit.trace(lambda x: ops.dispatch(x, order), x, check_trace=False)


def test_a_gradient_from_what_out_held_is_refused():
    g = many._gen(95)
    lin = ops.Linear8(many._whole(g, 24, 32), torch.rand(24, device=DEV, generator=g))
    x, factor = many._randn(g, 7, 32).to(BF16), torch.ones((), dtype=BF16, device=DEV)
    out = lin(x)
    product = out * factor.requires_grad_()
    lin(x, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()

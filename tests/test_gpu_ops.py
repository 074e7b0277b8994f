"""Routing, experts and adapters (vllm_expert_cache/ops.py) on the GPU against their formulas in
64 bits.

Tolerances. An output is off by half a step of its type (2^-8 of the value for bfloat16, 2^-11
for float16) and by what 32-bit sums leave: a sum of K products is off by at most
gamma(K) = 2 * K * 2^-24 of the sum of their absolute values (twice the classical bound, since
the matrix cores' order and rounding are their own). Values split into two bfloat16 are off by
2^-16. `_moe` and `_adapt` carry those bounds through the formulas beside the values.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import gpu_util as gu
from vllm_expert_cache import ops
from vllm_expert_cache.cache import ExpertSlotCache

pytestmark = pytest.mark.gpu

DEV = gu.DEV
BF16, F16, F32, I8, E4 = (torch.bfloat16, torch.float16, torch.float32, torch.int8,
                          torch.float8_e4m3fn)
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {BF16: 2.0 ** -126, F16: 2.0 ** -24}
SPLIT = 2.0 ** -16


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _gamma(k):
    return 2 * k * 2.0 ** -24


def _close(got, want, bound):
    """|got - want| <= bound where `want` is finite; the same infinity or NaN elsewhere."""
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    off = ((got - want).abs() - bound)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, \
        f"off by {float((got - want).abs()[fine].max())}, {float(off.max())} over the bound"


# ---- experts ------------------------------------------------------------------------------

def _weights(g, S, rows, cols, kind):
    v = torch.randn((S, rows, cols), device=DEV, generator=g)
    if kind == I8:
        return (v * 40).round().clamp(-128, 127).to(I8), \
            (0.5 + torch.rand((S, rows), device=DEV, generator=g)) * cols ** -0.5 / 40
    if kind == E4:
        shape = (S, -(-rows // 128), -(-cols // 128))
        return (v * 60).clamp(-448, 448).to(E4), \
            (0.5 + torch.rand(shape, device=DEV, generator=g)) * cols ** -0.5 / 60
    return (v * cols ** -0.5).to(kind), None


def _whole(w, scale):
    v = w.double()
    if scale is None:
        return v
    if w.dtype == I8:
        return v * scale.double().view(-1, 1)
    full = torch.kron(scale.double(), torch.ones(128, 128, dtype=torch.float64, device=DEV))
    return v * full[:v.shape[0], :v.shape[1]]


def _moe(e, x, probs, ids):
    """(output, bound on its error) by the formula in 64 bits."""
    T, H = x.shape
    y = torch.zeros((T, H), dtype=torch.float64, device=DEV)
    err = torch.zeros_like(y)
    xd, I = x.double(), e.I
    for t in range(T):
        for j in range(ids.shape[1]):
            s, p = int(ids[t, j]), float(probs[t, j])
            if not 0 <= s < e.S or p == 0:
                continue
            w13 = _whole(e.w13[s], None if e.w13_scale is None else e.w13_scale[s])
            w2 = _whole(e.w2[s], None if e.w2_scale is None else e.w2_scale[s])
            gu_, size = (w13 * xd[t]).sum(1), (w13 * xd[t]).abs().sum(1)
            g, u = gu_[:I], gu_[I:]
            act = g * torch.sigmoid(g)
            h = act * u
            dg, du = _gamma(H + 8) * size[:I], _gamma(H + 8) * size[I:]
            dh = 1.1 * dg * u.abs() + act.abs() * du + dg * du + 16 * 2.0 ** -24 * h.abs()
            y[t] += (w2 * (h * p)).sum(1)
            err[t] += ((w2.abs() * (dh * abs(p))).sum(1) +
                       (_gamma(2 * I + 80) + SPLIT) * (w2 * (h * p)).abs().sum(1))
    return y, err * 1.01 + HALF[x.dtype] * (y.abs() + err) + TINY[x.dtype]


def _experts(seed, S, H, I, kind):
    g = _gen(seed)
    w13, s13 = _weights(g, S, 2 * I, H, kind)
    w2, s2 = _weights(g, S, H, I, kind)
    return ops.Experts(w13, w2, s13, s2)


def _tokens(seed, T, k, S, H, dtype, id_dtype=torch.int32):
    g = _gen(seed + 1)
    x = torch.randn((T, H), device=DEV, generator=g).to(dtype)
    probs = torch.softmax(torch.randn((T, k), device=DEV, generator=g), 1)
    ids = torch.rand((T, S), device=DEV, generator=g).topk(min(k, S), 1).indices
    ids = ids.repeat(1, -(-k // S))[:, :k].to(id_dtype).contiguous()
    return x, probs, ids


KINDS = [(BF16, BF16), (F16, F16), (BF16, I8), (F16, I8), (BF16, E4), (F16, E4)]
# tokens, top_k, slots, hidden, inter: one pair; lengths below, at and past a unit of 128 and
# with tails; more than one tile of 16 tokens an expert; more pairs than slots
SHAPES = [(1, 1, 1, 16, 16), (1, 2, 4, 128, 128), (2, 4, 6, 272, 144), (5, 3, 3, 400, 48),
          (16, 8, 20, 144, 272), (17, 2, 5, 128, 64), (40, 1, 1, 160, 80), (33, 5, 37, 64, 32)]


@pytest.mark.parametrize("T,k,S,H,I", SHAPES)
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_experts(T, k, S, H, I, dtype, kind):
    e = _experts(T * 100 + H, S, H, I, kind)
    x, probs, ids = _tokens(T, T, k, S, H, dtype, torch.int64 if T % 2 else torch.int32)
    _close(e(x, probs, ids), *_moe(e, x, probs, ids))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("H,I", [(8, 8), (24, 40), (136, 24), (520, 136)])
def test_experts_rows_that_end_inside_a_tile(dtype, H, I):
    e = _experts(H, 4, H, I, dtype)
    x, probs, ids = _tokens(H, 3, 2, 4, H, dtype)
    _close(e(x, probs, ids), *_moe(e, x, probs, ids))


@pytest.mark.parametrize("kind", [I8, E4, BF16, F16])
@pytest.mark.parametrize("T,k,S,H,I", [(17, 2, 40, 256, 512), (20, 2, 60, 192, 784),
                                       (33, 1, 30, 64, 144)])
def test_experts_of_one_or_two_tokens_among_many(T, k, S, H, I, kind):
    """Many tokens over more slots: each expert has a token or two, and lengths of several units
    that end whole or inside one."""
    e = _experts(T + I, S, H, I, kind)
    x, probs, ids = _tokens(T + H, T, k, S, H, F16 if kind == F16 else BF16)
    _close(e(x, probs, ids), *_moe(e, x, probs, ids))


@pytest.mark.parametrize("T,k,S", [(16, 64, 70), (64, 16, 9), (1024, 1, 3), (1, 64, 64)])
def test_experts_largest_calls(T, k, S):
    e = _experts(T, S, 48, 32, BF16)
    x, probs, ids = _tokens(T, T, k, S, 48, BF16)
    _close(e(x, probs, ids), *_moe(e, x, probs, ids))


@pytest.mark.parametrize("T,S", [(3, 8), (20, 8), (1, 2)])
def test_experts_pairs_that_add_nothing(T, S):
    """Ids outside the slots, zero weights, tokens with neither, and the same slot twice."""
    e = _experts(T, S, 64, 48, BF16)
    x, probs, ids = _tokens(T, T, 4, S, 64, BF16, torch.int64)
    ids[:, 1] = ids[:, 0]                      # twice the same slot
    ids[0, 2], ids[0, 3] = -1, S
    ids[-1, 3] = 2 ** 32 + 1                   # not slot 1
    probs[T // 2, 2] = 0.0
    if T > 2:
        ids[1] = -5
        probs[2] = 0.0
    y = e(x, probs, ids)
    _close(y, *_moe(e, x, probs, ids))
    if T > 2:
        assert not y[1].any() and not y[2].any()
    assert not e(x, torch.zeros_like(probs), ids).any()
    assert e(x[:0], probs[:0], ids[:0]).shape == (0, 64)


@pytest.mark.parametrize("kind", [BF16, F16, E4])
@pytest.mark.parametrize("T", [4, 30])
def test_experts_numbers_that_are_none_stay_where_they_belong(kind, T):
    """NaN and infinity in an expert or a token reach the tokens that are routed to it alone."""
    dtype = F16 if kind == F16 else BF16
    H = 160
    e = _experts(3, 6, H, 48, kind)
    x, probs, ids = _tokens(9, T, 2, 4, H, dtype)   # slots 4 and 5 are nobody's
    clean = e(x, probs, ids)
    bad = float("nan") if kind == E4 else float("inf")
    for w in (e.w13, e.w2):
        w[4], w[5] = torch.full_like(w[4], 1.0), torch.full_like(w[5], bad)
    assert torch.equal(e(x, probs, ids), clean)
    ids2, probs2 = ids.clone(), probs.clone()
    ids2[0, 0], probs2[0, 0] = 5, 0.0                # weight 0: left out, whatever it holds
    want, bound = _moe(e, x, probs2, ids2)
    _close(e(x, probs2, ids2), want, bound)
    ids2[1, 0] = 5
    got = e(x, probs2, ids2)
    assert not torch.isfinite(got[1]).any()
    # the other tokens' sums may have another order: the formula's bound holds for any
    _close(got[2:], want[2:], bound[2:])
    x2 = x.clone()
    x2[2, 7] = float("nan")
    got = e(x2, probs, ids)
    assert torch.isnan(got[2]).all()
    rest = [t for t in range(T) if t != 2]
    want, bound = _moe(e, x, probs, ids)
    _close(got[rest], want[rest], bound[rest])


def test_experts_hidden_values_past_float16():
    """Hidden values over 65504 with float16 tokens and weights."""
    g = _gen(4)
    w13 = (torch.randn((2, 64, 32), device=DEV, generator=g) * 30).to(F16)
    w2 = (torch.randn((2, 32, 32), device=DEV, generator=g) * 2.0 ** -14).to(F16)
    e = ops.Experts(w13, w2)
    x, probs, ids = _tokens(5, 3, 2, 2, 32, F16)
    x = x * 4
    y, bound = _moe(e, x, probs, ids)
    hidden = (w13[0].double() @ x[0].double())
    assert float((hidden[:32] * hidden[32:]).abs().max()) > 65504
    _close(e(x, probs, ids), y, bound)


@pytest.mark.parametrize("dtype,kind", [(BF16, BF16), (F16, I8)])
def test_experts_strides_and_out(dtype, kind):
    """Tokens that are columns of a wider tensor, at an odd stride and at an odd address; a
    strided `out` whose other columns stay."""
    H = 96
    e = _experts(8, 5, H, 64, kind)
    x, probs, ids = _tokens(8, 6, 3, 5, H, dtype)
    want = e(x, probs, ids)
    for pad, at in ((8, 8), (32, 0), (5, 3), (1, 1)):
        wide = torch.zeros((6, H + pad), dtype=dtype, device=DEV)
        wide[:, at:at + H] = x
        assert torch.equal(e(wide[:, at:at + H], probs, ids), want)
        assert torch.equal(e(wide[2:3, at:at + H], probs[2:3], ids[2:3]), want[2:3])
        out = torch.full((6, H + pad), 7.0, dtype=dtype, device=DEV)
        assert e(x, probs, ids, out=out[:, at:at + H]).data_ptr() == out[:, at:].data_ptr()
        assert torch.equal(out[:, at:at + H], want)
        assert (out[:, :at] == 7).all() and (out[:, at + H:] == 7).all()
    flipped = probs.t().contiguous().t()
    assert torch.equal(e(x, flipped, ids.t().contiguous().t()), want)


def test_experts_do_not_depend_on_the_batch():
    """A token's result is the same alone and in a batch of up to 16 tokens, and in each call."""
    e = _experts(2, 12, 256, 128, I8)
    x, probs, ids = _tokens(2, 16, 4, 12, 256, BF16)
    y = e(x, probs, ids)
    for _ in range(3):
        assert torch.equal(e(x, probs, ids), y)
    _close(torch.cat([e(x[t:t + 1], probs[t:t + 1], ids[t:t + 1]) for t in range(16)]),
           *_moe(e, x, probs, ids))


def test_experts_offsets_past_32_bits():
    """Slabs of 2^29 weights and more: the last slot starts past 2^31 elements."""
    S, H, I = 6, 16384, 13120   # w13 429,916,160 elements a slot
    w13 = torch.zeros((S, 2 * I, H), dtype=I8, device=DEV)
    w2 = torch.zeros((S, H, I), dtype=I8, device=DEV)
    g = _gen(1)
    small, s13 = _weights(g, 1, 2 * I, 64, I8)
    down, s2 = _weights(g, 1, 64, I, I8)
    w13[S - 1, :, -64:] = small[0]
    w2[S - 1, -64:] = down[0]
    assert (S - 1) * 2 * I * H > 2 ** 31
    s13 = s13.expand(S, -1).contiguous()
    s2 = torch.cat([torch.ones((1, H - 64), device=DEV), s2], 1).expand(S, -1).contiguous()
    e = ops.Experts(w13, w2, s13, s2)
    x = torch.randn((2, H), device=DEV, generator=g).to(BF16)
    ids = torch.tensor([[S - 1], [0]], device=DEV)
    probs = torch.ones((2, 1), device=DEV)
    got = e(x, probs, ids)
    assert not got[1].any() and not got[0, :-64].any()
    gu_ = (small[0].double() * s13[0].double()[:, None]) @ x[0, -64:].double()
    h = gu_[:I] * torch.sigmoid(gu_[:I]) * gu_[I:]
    terms = down[0].double() * s2[0, -64:].double()[:, None] * h
    bound = (_gamma(2 * I) + SPLIT + 4 * _gamma(64)) * 4 * terms.abs().sum(1)
    want = terms.sum(1)
    _close(got[0, -64:], want, bound + HALF[BF16] * want.abs())


# ---- adapters -----------------------------------------------------------------------------

def _adapt(l, x, base, ids):
    T = x.shape[0]
    y, err = base.double().clone(), torch.zeros(base.shape, dtype=torch.float64, device=DEV)
    for t in range(T):
        s = int(ids[t])
        if not 0 <= s < l.S:
            continue
        a, b = l.a[s].double(), l.b[s].double()
        f = 1.0 if l.scales is None else float(l.scales[s])
        v, size = (a * x[t].double()).sum(1), (a * x[t].double()).abs().sum(1)
        y[t] += (b * v).sum(1) * f
        err[t] = abs(f) * ((b.abs() * size).sum(1) * _gamma(l.H + 16) +
                           (b * v).abs().sum(1) * (_gamma(2 * l.R + 8) + SPLIT))
    return y, err * 1.01 + HALF[x.dtype] * (y.abs() + err) + TINY[x.dtype]


def _adapters(seed, S, R, H, O, dtype, scaled=True):
    g = _gen(seed)
    return ops.Adapters(
        (torch.randn((S, R, H), device=DEV, generator=g) * H ** -0.5).to(dtype),
        (torch.randn((S, O, R), device=DEV, generator=g) * R ** -0.5).to(dtype),
        0.5 + torch.rand(S, device=DEV, generator=g) if scaled else None)


def _adapter_tokens(seed, T, S, H, O, dtype, run, id_dtype=torch.int32):
    """Tokens whose adapter changes about every `run` tokens; one in nine has none."""
    g = _gen(seed)
    x = torch.randn((T, H), device=DEV, generator=g).to(dtype)
    base = torch.randn((T, O), device=DEV, generator=g).to(dtype)
    turn = (torch.rand(T, device=DEV, generator=g) < 1 / run).long().cumsum(0)
    slot = torch.randint(0, S, (T + 1,), device=DEV, generator=g)
    slot[torch.rand(T + 1, device=DEV, generator=g) < 1 / 9] = -1
    return x, base, slot[turn].to(id_dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,run,S,R,H,O", [
    (1, 1, 1, 8, 8, 1), (1, 1, 4, 16, 256, 64), (3, 1, 8, 8, 128, 17), (16, 1, 32, 32, 264, 130),
    (17, 2, 5, 24, 520, 63), (50, 9, 6, 64, 1048, 96), (200, 40, 3, 40, 64, 256),
    (33, 1, 64, 256, 136, 48), (5, 1, 5, 16, 4104, 8),
    (7, 2, 4, 48, 72, 40), (16, 1, 20, 72, 136, 33), (40, 3, 9, 136, 200, 70)])
def test_adapters(dtype, T, run, S, R, H, O):
    l = _adapters(T + R, S, R, H, O, dtype, scaled=T % 2 == 1)
    x, base, ids = _adapter_tokens(T, T, S, H, O, dtype, run,
                                   torch.int64 if S % 2 else torch.int32)
    kept = base.clone()
    y = l(x, base, ids)
    assert torch.equal(base, kept)
    _close(y, *_adapt(l, x, base, ids))
    assert l(x, base, ids, out=base) is base   # in place
    assert torch.equal(base, y)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,run,S,R,H,O", [
    (129, 200, 2, 8, 8, 1), (150, 1, 70, 24, 136, 33), (193, 30, 4, 64, 392, 514),
    (300, 100, 3, 72, 1032, 127), (257, 60, 5, 256, 264, 65), (1000, 300, 2, 16, 2056, 72),
    (280, 1, 70, 24, 136, 33), (257, 30, 4, 8, 8, 1), (321, 30, 4, 64, 392, 514)])
def test_adapters_of_many_tokens(dtype, T, run, S, R, H, O):
    """Many tokens: long runs of an adapter and tokens that all differ, ranks of one, two and
    more tiles, ends inside tiles, odd addresses, in place, rows without an adapter."""
    l = _adapters(T + R, S, R, H, O, dtype, scaled=T % 2 == 1)
    x, base, ids = _adapter_tokens(T + 1, T, S, H, O, dtype, run,
                                   torch.int64 if S % 2 else torch.int32)
    ids[T // 2], ids[T - 1] = -1, S            # none, in the middle of a run and at the end
    y = l(x, base, ids)
    _close(y, *_adapt(l, x, base, ids))
    for t in (T // 2, T - 1):
        assert torch.equal(y[t], base[t])
    wx = torch.full((T, H + 5), float("nan"), dtype=dtype, device=DEV)
    wb = torch.full((T, O + 3), 5.0, dtype=dtype, device=DEV)
    wx[:, 3:H + 3], wb[:, 1:O + 1] = x, base
    view = wb[:, 1:O + 1]
    assert l(wx[:, 3:H + 3], view, ids, out=view) is view
    assert torch.equal(view, y)
    assert (wb[:, :1] == 5).all() and (wb[:, O + 1:] == 5).all()


def test_adapters_of_many_tokens_keep_what_is_no_number_apart():
    l = _adapters(11, 5, 40, 200, 70, BF16)
    x, base, ids = _adapter_tokens(11, 260, 4, 200, 70, BF16, 25)
    clean = l(x, base, ids)
    l.a[4], l.b[4] = float("inf"), float("nan")     # nobody's
    assert torch.equal(l(x, base, ids), clean)
    ids[7], ids[130] = 4, -1
    x[9, 3] = x[130, 5] = float("nan")
    ids[9] = 1
    base[200, 4] = float("inf")
    got = l(x, base, ids)
    assert torch.isnan(got[7]).all() and torch.isnan(got[9]).all()
    assert torch.equal(got[130], base[130]) and got[200, 4] == float("inf")
    rest = [t for t in range(260) if t not in (7, 9, 130, 200)]
    _close(got[rest], *(v[rest] for v in _adapt(l, torch.nan_to_num(x), base, ids.clamp(max=3))))


def test_adapters_rows_without_one_stay_as_they_are():
    l = _adapters(3, 4, 16, 64, 40, BF16)
    x, base, ids = _adapter_tokens(3, 20, 4, 64, 40, BF16, 1, torch.int64)
    ids[2], ids[3], ids[4], ids[5] = -1, 4, -2 ** 40, 2 ** 32
    base[2], base[5] = float("nan"), float("inf")
    x[3] = float("nan")                        # a token without an adapter is not read for one
    y = l(x, base, ids)
    for t in (2, 3, 4, 5):
        assert torch.equal(y[t].view(torch.int16), base[t].view(torch.int16))
    x[3] = 0
    ok = [t for t in range(20) if t not in (2, 5)]
    want, bound = _adapt(l, x, base, ids)
    _close(y[ok], want[ok], bound[ok])
    none = torch.full((20,), -1, device=DEV)
    assert torch.equal(l(x, base, none).view(torch.int16), base.view(torch.int16))
    assert l(x[:0], base[:0], ids[:0]).shape == (0, 40)


def test_adapters_numbers_that_are_none_stay_where_they_belong():
    l = _adapters(5, 5, 16, 96, 48, BF16)
    x, base, ids = _adapter_tokens(5, 24, 4, 96, 48, BF16, 1)
    clean = l(x, base, ids)
    l.a[4], l.b[4] = float("inf"), float("nan")     # nobody's
    assert torch.equal(l(x, base, ids), clean)
    ids[7] = 4
    x[9, 3] = float("nan")
    ids[9] = 1
    got = l(x, base, ids)
    assert torch.isnan(got[7]).all() and torch.isnan(got[9]).all()
    rest = [t for t in range(24) if t not in (7, 9)]
    assert torch.equal(got[rest], clean[rest])


def test_adapters_strides():
    l = _adapters(6, 4, 24, 72, 33, F16)
    x, base, ids = _adapter_tokens(6, 19, 4, 72, 33, F16, 3)
    want = l(x, base, ids)
    for pad, at in ((8, 8), (5, 3), (3, 0)):
        wx = torch.zeros((19, 72 + pad), dtype=F16, device=DEV)
        wb = torch.full((19, 33 + pad), 5.0, dtype=F16, device=DEV)
        wx[:, at:at + 72], wb[:, at:at + 33] = x, base
        assert torch.equal(l(wx[:, at:at + 72], wb[:, at:at + 33], ids), want)
        assert torch.equal(l(wx[4:5, at:at + 72], wb[4:5, at:at + 33], ids[4:5]), want[4:5])
        view = wb[:, at:at + 33]
        l(x, view, ids, out=view)
        assert torch.equal(view, want)
        assert (wb[:, :at] == 5).all() and (wb[:, at + 33:] == 5).all()
    shared = base[:1].expand(19, 33)                # one row for all
    assert torch.equal(l(x, shared, ids), l(x, shared.contiguous(), ids))


def test_adapters_offsets_past_32_bits():
    S, R, H, O = 1030, 256, 8192, 16
    a = torch.zeros((S, R, H), dtype=BF16, device=DEV)
    b = torch.zeros((S, O, R), dtype=BF16, device=DEV)
    g = _gen(2)
    a[-1] = torch.randn((R, H), device=DEV, generator=g) * H ** -0.5
    b[-1] = torch.randn((O, R), device=DEV, generator=g) / 16
    assert (S - 1) * R * H > 2 ** 31
    l = ops.Adapters(a, b)
    x, base, _ = _adapter_tokens(1, 3, 1, H, O, BF16, 1)
    ids = torch.tensor([S - 1, 0, S - 1], device=DEV)
    _close(l(x, base, ids), *_adapt(l, x, base, ids))


# ---- routing ------------------------------------------------------------------------------

def _route(logits, k, scoring="softmax", bias=None, groups=1, topk_groups=1, renormalize=True,
           scale=1.0):
    """Row by row from the definition, in numpy's 64 bits."""
    x = logits.float().cpu().numpy().astype(np.float64)
    b = None if bias is None else bias.cpu().numpy().astype(np.float64)
    T, E = x.shape
    w, ids = np.zeros((T, k)), np.full((T, k), -1)
    for t in range(T):
        live = [e for e in range(E) if x[t, e] > -np.inf and (b is None or b[e] > -np.inf)]
        seen = [e for e in range(E) if x[t, e] > -np.inf]
        if not live:
            continue
        top = max(x[t, e] for e in seen)
        part = {e: 1.0 if x[t, e] == top else math.exp(x[t, e] - top) for e in seen}
        total = sum(part.values())
        score = {e: part[e] / total if scoring == "softmax" else
                 1 / (1 + math.exp(-x[t, e])) if x[t, e] > -700 else 0.0 for e in live}
        key = {e: x[t, e] if b is None else score[e] + b[e] for e in live}
        n = E // groups
        if groups > 1:
            worth = {}
            for g in range(groups):
                best = sorted((key[e] for e in live if e // n == g), reverse=True)
                if best:
                    worth[g] = sum(best[:2]) if b is not None else best[0]
            kept = sorted(worth, key=lambda g: (-worth[g], g))[:topk_groups]
            live = [e for e in live if e // n in kept]
        chosen = sorted(live, key=lambda e: (-key[e], e))[:k]
        s = sum(score[e] for e in chosen)
        for j, e in enumerate(chosen):
            ids[t, j] = e
            w[t, j] = scale * (score[e] / s if renormalize and s > 0 else
                               0.0 if renormalize else score[e])
    return w, ids


def _check_route(logits, k, **kw):
    w, ids = ops.route(logits, k, **kw)
    kw.pop("id_dtype", None)
    want_w, want_ids = _route(logits, k, **kw)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    # every weight is made in 64 bits and rounded once
    np.testing.assert_allclose(w.cpu().numpy(), want_w, rtol=1.01 * 2.0 ** -24, atol=1e-38)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 128, 8), (3, 8, 8), (5, 64, 6), (7, 65, 10),
                                   (9, 200, 1), (4, 257, 33), (6, 512, 64), (5, 1000, 12),
                                   (2, 1024, 64)])
def test_route(dtype, T, E, k):
    logits = (2 * torch.randn((T, E), device=DEV, generator=_gen(E))).to(dtype)
    bias = 0.2 * torch.randn(E, device=DEV, generator=_gen(k))
    _check_route(logits, k)
    _check_route(logits, k, scoring="sigmoid", renormalize=False, scale=2.5, id_dtype=torch.int64)
    _check_route(logits, k, bias=bias, renormalize=False)
    _check_route(logits, k, bias=bias, scoring="sigmoid", scale=1.5)


@pytest.mark.parametrize("E,groups,topk_groups,k", [
    (8, 8, 3, 3), (16, 4, 2, 5), (64, 8, 4, 8), (256, 8, 4, 8), (130, 5, 2, 9), (96, 3, 1, 4),
    (512, 64, 7, 20), (192, 2, 2, 6), (1024, 16, 5, 16), (66, 33, 10, 7)])
def test_route_groups(E, groups, topk_groups, k):
    logits = 2 * torch.randn((9, E), device=DEV, generator=_gen(E + k))
    bias = 0.3 * torch.randn(E, device=DEV, generator=_gen(k))
    kw = dict(groups=groups, topk_groups=topk_groups)
    _check_route(logits, k, **kw)
    _check_route(logits, k, bias=bias, scoring="sigmoid", **kw)
    logits[1, :E // groups] = -math.inf          # a group that is masked out
    logits[2, 1:E // groups] = -math.inf         # one expert of a group left
    logits[3] = -math.inf                        # nothing left
    logits[4, k // 2:] = -math.inf               # fewer left than asked for
    _check_route(logits, k, **kw)
    _check_route(logits, k, bias=bias, scoring="sigmoid", renormalize=False, **kw)


def test_route_ties_masks_and_no_numbers():
    inf, nan = math.inf, math.nan
    E = 70
    rows = torch.zeros((12, E))
    rows[1, ::2] = -0.0                          # -0 and 0 are equal
    rows[2] = torch.arange(E) // 3               # threes
    rows[3] = -inf
    rows[4, 3:] = -inf
    rows[5, 10] = rows[5, 66] = inf              # the infinite ones share
    rows[6, 5] = nan
    rows[7] = nan
    rows[8] = -3.4e38                            # a mask of the type's lowest value
    rows[8, 40] = 1.0
    rows[9] = 60.0 + torch.arange(E) % 2         # sigmoids of 1, softmax of steps
    rows[10] = -90.0 - torch.arange(E) % 2
    rows[11] = torch.linspace(-1e-3, 1e-3, E)
    rows = rows.to(DEV)
    for k in (1, 6, 20):
        _check_route(rows, k)
        _check_route(rows, k, renormalize=False)
        _check_route(rows, k, scoring="sigmoid")
        _check_route(rows, k, bias=torch.zeros(E, device=DEV))
        bias = torch.zeros(E, device=DEV)
        bias[2], bias[3], bias[4] = -inf, nan, 1e30
        _check_route(rows[:9], k, bias=bias, scoring="sigmoid")
        _check_route(rows, k, groups=7, topk_groups=3)


def test_route_many_tokens_and_strides():
    logits = torch.randn((4099, 128), device=DEV, generator=_gen(1)).to(BF16)
    w, ids = ops.route(logits, 8)
    order = logits.double().sort(dim=1, descending=True, stable=True).indices[:, :8]
    assert torch.equal(ids.long(), order)
    want = torch.softmax(logits.double().gather(1, order), 1)
    assert float((w.double() - want).abs().max()) <= 2.0 ** -25
    wide = torch.randn((9, 133), device=DEV, generator=_gen(2))
    _check_route(wide[:, 3:70], 5)
    _check_route(wide.t()[:67].t(), 5)
    _check_route(wide[:1].expand(9, 133), 5)
    assert ops.route(wide[:0], 5)[1].shape == (0, 5)


# ---- together -----------------------------------------------------------------------------

class _Owner:
    pass


def _host(t):
    out = torch.empty(t.shape, dtype=t.dtype, pin_memory=True)
    out.copy_(t)
    return out


@pytest.mark.parametrize("kind", [BF16, I8, E4])
def test_a_layer_from_logits_to_hidden_states_through_the_cache(kind):
    """route, refresh and the experts over the cache's slots, step after step with the experts
    in host memory: the same as the experts read whole."""
    E, S, H, I, k, T = 24, 8, 128, 64, 2, 3
    g = _gen(7)
    w13, s13 = _weights(g, E, 2 * I, H, kind)
    w2, s2 = _weights(g, E, H, I, kind)
    whole = ops.Experts(w13, w2, s13, s2)
    owner = _Owner()
    owner.w13_weight, owner.w2_weight = _host(w13), _host(w2)
    names = ["w13_weight", "w2_weight"]
    if s13 is not None:
        pad = (lambda s: s) if kind == I8 else (lambda s: s.reshape(E, -1).repeat(1, 4))
        owner.s13, owner.s2 = _host(pad(s13)), _host(pad(s2))
        names += ["s13", "s2"]
    cache = ExpertSlotCache(owner, names, E, S, DEV, required=names[:2])
    for t in cache.slots.values():
        t.zero_()
    scales = ()
    if kind == I8:
        scales = (cache.slots["s13"], cache.slots["s2"])
    elif kind == E4:   # one block each at this size, four times to make 16 bytes
        scales = tuple(cache.slots[n][:, :s[0].numel()].reshape(S, *s.shape[1:]).contiguous()
                       for n, s in (("s13", s13), ("s2", s2)))
    slots = ops.Experts(cache.slots["w13_weight"], cache.slots["w2_weight"], *scales)
    gate = torch.randn((E, H), device=DEV, generator=g)
    for step in range(20):
        x = torch.randn((T, H), device=DEV, generator=g).to(BF16)
        weights, ids = ops.route(x.float() @ gate.t(), k)
        at = cache.refresh(ids)
        if kind == E4:
            for n, s, mine in (("s13", s13, slots.w13_scale), ("s2", s2, slots.w2_scale)):
                mine.copy_(cache.slots[n][:, :s[0].numel()].reshape(mine.shape))
        assert torch.equal(slots(x, weights, at), whole(x, weights, ids)), step


def test_adapters_through_the_cache():
    """Adapters of more requests than there are slots, brought in by refresh."""
    N, S, R, H, O = 40, 12, 16, 128, 96
    whole = _adapters(11, N, R, H, O, BF16)
    owner = _Owner()
    owner.a, owner.b = _host(whole.a), _host(whole.b)
    cache = ExpertSlotCache(owner, ["a", "b"], N, S, DEV)
    slots = ops.Adapters(cache.slots["a"], cache.slots["b"])
    plain = ops.Adapters(whole.a, whole.b)
    rng = np.random.default_rng(3)
    for step in range(12):
        requests = torch.as_tensor(rng.choice(N, 9, replace=False).astype(np.int32), device=DEV)
        token_of = torch.as_tensor(np.sort(rng.integers(0, 9, 30)), device=DEV)
        x, base, _ = _adapter_tokens(step, 30, S, H, O, BF16, 1)
        at = cache.refresh(requests)
        got = slots(x, base, at[token_of])
        assert torch.equal(got, plain(x, base, requests[token_of])), step


def _everything():
    g = _gen(21)
    e = _experts(21, 12, 256, 128, I8)
    l = _adapters(21, 12, 16, 256, 256, BF16)
    logits = torch.randn((5, 12), device=DEV, generator=g).to(BF16)
    x = torch.randn((5, 256), device=DEV, generator=g).to(BF16)
    ids = torch.tensor([0, 3, -1, 3, 7], device=DEV)

    def step():
        w, experts = ops.route(logits, 3)
        return l(x, e(x, w, experts), ids)

    return logits, x, step


def test_captured_and_replayed():
    """A graph of the three, replayed on new inputs with eager calls and synchronisations
    between, and a second graph beside it."""
    logits, x, step = _everything()
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(6):
        x.copy_(torch.randn(x.shape, device=DEV, generator=_gen(i)))
        logits.copy_(torch.randn(logits.shape, device=DEV, generator=_gen(50 + i)))
        for graph, _ in graphs:
            graph.replay()
        want = step()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want), i


def test_two_streams_at_once():
    _, _, first = _everything()
    _, _, second = _everything()
    want = first()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, (s, step) in enumerate(zip(streams, (first, second))):
            with torch.cuda.stream(s):
                got[i].append(step())
    torch.cuda.synchronize()
    for outs in got:
        for o in outs:
            assert torch.equal(o, want)


@pytest.mark.parametrize("T", [20, 300])
def test_many_tokens_captured_and_on_two_streams(T):
    """The launches of more than 16 tokens of experts and more than 256 of adapters: replayed on
    new inputs, and two at once. The last tokens are padding: no ids, and x that is no number."""
    S, H, k = 12, 256, 3
    e, l = _experts(T, S, H, 128, E4), _adapters(T, S, 24, H, H, BF16)
    x, probs, ids = _tokens(T, T, k, S, H, BF16)
    _, base, slots = _adapter_tokens(T, T, S, H, H, BF16, 30)
    pad = T - 4
    ids[pad:], slots[pad:], x[pad:] = -1, -1, float("nan")

    def step():
        return l(x, base, slots), e(x, probs, ids)

    def check(got):
        low, y = got
        _close(low[:pad], *(v[:pad] for v in _adapt(l, x, base, slots)))
        _close(y[:pad], *(v[:pad] for v in _moe(e, torch.nan_to_num(x), probs, ids)))
        assert torch.equal(low[pad:], base[pad:]) and not y[pad:].any()

    check(step())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x[:pad].copy_(torch.randn((pad, H), device=DEV, generator=_gen(i)))
        probs.copy_(torch.rand((T, k), device=DEV, generator=_gen(50 + i)))
        ids[:pad] = ids[:pad].flip(0)
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        check(out)
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), i
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    for pair in got:
        assert all(torch.equal(a, b) for a, b in zip(pair, out))

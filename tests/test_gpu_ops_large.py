"""The operators' kernels on lengths and calls where every loop of theirs runs full: several units
of 128 a wave or workgroup, 8 and 16 rows a workgroup, waves that share a length and waves that do
not, against the formulas in 64 bits.

What goes into the first products is a small multiple of a power of two, so their sums are exact in
32 bits in any order, and a unit left out or taken twice shows in full: the bound on an output is
what the rest of the formula leaves (test_gpu_ops.py says how): 16 * 2^-24 for SiLU, product and
weight, gamma of the second products' length, SPLIT for values in two bfloat16, and half a step of
the output's type.
"""
from __future__ import annotations

import pytest
import torch

import gpu_util as gu
from test_gpu_ops import (BF16, E4, F16, HALF, I8, KINDS, SPLIT, TINY, _adapter_tokens, _close,
                          _gamma, _gen, _tokens, _weights, _whole)
from vllm_expert_cache import ops

pytestmark = pytest.mark.gpu

DEV = gu.DEV


def _small(g, shape, most, dtype, unit=1.0):
    return (torch.randint(-most, most + 1, shape, device=DEV, generator=g) * unit).to(dtype)


def _powers(g, shape, low):
    """2^low or twice that."""
    return torch.randint(1, 3, shape, device=DEV, generator=g).float() * 2.0 ** low


def _experts(seed, S, H, I, kind):
    """w13 of at most 6 * 2^-6: a sum over H of products with whole numbers of at most 2 is at most
    12 * H steps of 2^-6, fewer than 2^24 up to an H of 2^20."""
    g = _gen(seed)
    if kind == I8:
        w13, s13 = _small(g, (S, 2 * I, H), 3, I8), _powers(g, (S, 2 * I), -6)
    elif kind == E4:
        w13 = torch.empty((S, 2 * I, H), dtype=E4, device=DEV)
        for s in range(S):
            w13[s] = _small(g, (2 * I, H), 3, torch.float32).to(E4)
        s13 = _powers(g, (S, -(-2 * I // 128), -(-H // 128)), -6)
    else:
        w13, s13 = _small(g, (S, 2 * I, H), 6, kind, 2.0 ** -6), None
    w2, s2 = _weights(g, S, H, I, kind)
    return ops.Experts(w13, w2, s13, s2)


def _moe(e, x, probs, ids):
    """(output, bound) of a layer whose gate and up sums are exact, slot by slot."""
    T, H = x.shape
    y = torch.zeros((T, H), dtype=torch.float64, device=DEV)
    size = torch.zeros_like(y)
    live = (probs != 0) & (ids >= 0) & (ids < e.S)
    for s in torch.unique(ids[live]).tolist():
        t, j = torch.nonzero((ids == s) & live, as_tuple=True)
        w13 = _whole(e.w13[s], None if e.w13_scale is None else e.w13_scale[s])
        w2 = _whole(e.w2[s], None if e.w2_scale is None else e.w2_scale[s])
        g, u = (x[t].double() @ w13.t().contiguous()).chunk(2, 1)
        h = g * torch.sigmoid(g) * u * probs[t, j].double()[:, None]
        y.index_add_(0, t, h @ w2.t().contiguous())
        size.index_add_(0, t, h.abs() @ w2.abs().t().contiguous())
    k = ids.shape[1]
    err = (16 * 2.0 ** -24 + _gamma(2 * e.I + 16 + k) + SPLIT) * size * 1.01
    return y, err + HALF[x.dtype] * (y.abs() + err) + TINY[x.dtype]


def _check(seed, T, k, S, H, I, dtype, kind):
    e = _experts(seed, S, H, I, kind)
    _, probs, ids = _tokens(seed, T, k, S, 8, dtype, torch.int64 if T % 2 else torch.int32)
    x = _small(_gen(seed + 2), (T, H), 2, dtype)
    _close(e(x, probs, ids), *_moe(e, x, probs, ids))


def _fit(length, kind):
    """`length` as one-byte weights take it."""
    return -(-length // 16) * 16 if kind in (I8, E4) else length


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("T,k,S,H,I", [
    (1, 2, 4, 4096, 1032),      # 16 rows a workgroup, two experts
    (4, 8, 20, 3992, 392),      # the same, an expert after another in a wave, a part of a tile
    (4, 8, 20, 4104, 392),      # 8 rows a workgroup
    (8, 2, 3, 4360, 264),       # two to four tokens an expert and more
    (1, 8, 16, 2040, 776),      # four units a wave up
    (8, 8, 24, 2056, 520),      # 16 rows again
    (2, 4, 6, 520, 4104),       # workgroups that share a length
    (16, 4, 12, 2056, 1032),    # nine and more tokens, at most 2^22 weights
])
def test_experts_of_few_tokens(dtype, kind, T, k, S, H, I):
    _check(T + H, T, k, S, _fit(H, kind), _fit(I, kind), dtype, kind)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("T,k,S,H,I", [
    (9, 2, 8, 4096, 1040),      # nine tokens, more than 2^22 weights: waves share the length
    (16, 4, 36, 4112, 1040),    # 36 experts: each wave has its own rows and all units
    (16, 5, 5, 2064, 2064),     # every token at every expert: a full tile of 16
    (64, 16, 600, 264, 392),    # 512 workgroups and more, a slot each, one or two tokens
    (128, 8, 1100, 264, 400),   # the same with a workgroup for every pair
    (200, 4, 20, 1032, 264),    # three tiles of tokens an expert
    (512, 2, 7, 392, 520),      # ten tiles
])
def test_experts_of_more_tokens(dtype, kind, T, k, S, H, I):
    _check(T + H, T, k, S, _fit(H, kind), _fit(I, kind), dtype, kind)


# ---- adapters -----------------------------------------------------------------------------

def _adapters(seed, S, R, H, O, dtype):
    g = _gen(seed)
    return ops.Adapters(_small(g, (S, R, H), 6, dtype, 2.0 ** -6),
                        (torch.randn((S, O, R), device=DEV, generator=g) * R ** -0.5).to(dtype),
                        0.5 + torch.rand(S, device=DEV, generator=g))


def _adapt(l, x, base, ids):
    """(output, bound) where A's sums are exact, slot by slot."""
    y, size = base.double().clone(), torch.zeros(base.shape, dtype=torch.float64, device=DEV)
    for s in torch.unique(ids[(ids >= 0) & (ids < l.S)]).tolist():
        t = torch.nonzero(ids == s)[:, 0]
        v = (x[t].double() @ l.a[s].double().t().contiguous()) * l.scales[s].double()
        b = l.b[s].double().t().contiguous()
        y.index_add_(0, t, v @ b)
        size.index_add_(0, t, v.abs() @ b.abs())
    err = (_gamma(2 * l.R + 8) + SPLIT) * size * 1.01
    return y, err + HALF[x.dtype] * (y.abs() + err) + TINY[x.dtype]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,run,S,R,H,O", [
    (2100, 25, 6, 72, 2056, 40),    # two or three units a workgroup
    (2100, 200, 6, 16, 4104, 136),  # four or five
    (4096, 30, 9, 64, 4096, 72),    # eight
    (4160, 90, 5, 136, 4104, 40),   # eight or nine, three lots of ranks
    (8200, 100, 4, 24, 4104, 24),   # 33, all of a row
])
def test_adapters_of_many_tokens(dtype, T, run, S, R, H, O):
    l = _adapters(T + R, S, R, H, O, dtype)
    _, base, ids = _adapter_tokens(T, T, S, 8, O, dtype, run)
    x = _small(_gen(T + 1), (T, H), 2, dtype)
    y = l(x, base, ids)
    _close(y, *_adapt(l, x, base, ids))
    none = ids < 0
    assert none.any() and torch.equal(y[none], base[none])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,run,S,R,H,O", [
    (1, 1, 2, 16, 65544, 72),    # one split a unit and wave
    (256, 3, 5, 8, 65544, 24),   # four units a wave, and five
    (250, 90, 3, 40, 81928, 8),
])
def test_adapters_of_long_rows(dtype, T, run, S, R, H, O):
    l = _adapters(T + R, S, R, H, O, dtype)
    _, base, ids = _adapter_tokens(T, T, S, 8, O, dtype, run)
    ids[0] = 1
    x = _small(_gen(T + 1), (T, H), 2, dtype)
    _close(l(x, base, ids), *_adapt(l, x, base, ids))

# ---- values of two bfloat16 ---------------------------------------------------------------

# 1 + 2^-8 is two bfloat16 (a tie: 1 and 2^-8), 1 + 7 * 2^-10 a float16 that is none. Eight of
# their products are 8 + 88 * 2^-10 + 56 * 2^-18, and ODD lifts that over the middle of two float16
# at 8 + 92 * 2^-10, which it does not reach without the last term. All products are multiples of
# 2^-18 and their sums below 2^4: exact in 32 bits in any order, so the result is exact, too.
LOW, ODD, WIDE, SUM = 1 + 2.0 ** -8, 2.0 ** -8 - 2.0 ** -13, 1 + 7 * 2.0 ** -10, 8 + 96 * 2.0 ** -10


@pytest.mark.parametrize("T", [1, 2, 20, 300])
def test_float16_experts_take_both_halves_of_a_value(T):
    w13 = torch.zeros((1, 64, 16), dtype=F16, device=DEV)
    w13[0, :9, 0] = 64.0                 # SiLU of 64 is 64 in 32 bits
    w13[0, 32:40, 1], w13[0, 40, 1] = LOW, ODD
    w2 = torch.zeros((1, 16, 32), dtype=F16, device=DEV)
    w2[0, :, :8], w2[0, :, 8] = WIDE, 1.0
    x = torch.zeros((T, 16), dtype=F16, device=DEV)
    x[:, :2] = 1.0
    y = ops.Experts(w13, w2)(x, torch.full((T, 1), 2.0 ** -6, device=DEV),
                             torch.zeros((T, 1), dtype=torch.int32, device=DEV))
    assert (y == SUM).all()


@pytest.mark.parametrize("T", [1, 20, 300])
def test_float16_adapters_take_both_halves_of_a_value(T):
    a = torch.eye(8, dtype=F16, device=DEV)[None].contiguous()
    b = torch.full((1, 24, 8), WIDE, dtype=F16, device=DEV)
    x = torch.full((T, 8), LOW, dtype=F16, device=DEV)
    base = torch.full((T, 24), ODD, dtype=F16, device=DEV)
    y = ops.Adapters(a, b)(x, base, torch.zeros(T, dtype=torch.int32, device=DEV))
    assert (y == SUM).all()

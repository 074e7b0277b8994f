"""What the operators say about inputs at their edges, each against values worked out here."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import gpu_util as gu
from test_gpu_ops import _close, _experts, _moe, _tokens
from vllm_expert_cache import ops

pytestmark = pytest.mark.gpu

DEV = gu.DEV
INF, NAN = math.inf, math.nan


# ---- routing ------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("none", [-INF, NAN])
@pytest.mark.parametrize("renormalize", [True, False])
def test_a_bias_that_excludes_an_expert_leaves_the_softmax_alone(dtype, none, renormalize):
    """Experts 0 and 65 are excluded, by a bias of -infinity or NaN: their logits still count in
    the softmax of the others."""
    E, k = 70, 5
    rows = torch.zeros((4, E))
    rows[0, 0], rows[0, 3], rows[0, 65] = 3.0, 2.0, 1.0
    rows[1] = torch.arange(E) / 16.0
    rows[1, 0] = 6.0                      # most of the row's weight
    rows[2, 1:] = -INF                    # nothing but an excluded one
    rows[3, 10:60] = NAN                  # no candidates and no part of the softmax
    rows = rows.to(dtype)
    bias = torch.zeros(E)
    bias[0], bias[65], bias[7] = none, none, 0.25
    w, ids = ops.route(rows.to(DEV), k, bias=bias.to(DEV), renormalize=renormalize)
    x = rows.double().numpy()
    e = np.where(np.isnan(x), 0.0, np.exp(np.where(np.isnan(x), 0, x) - np.nanmax(x, 1)[:, None]))
    score = e / e.sum(1, keepdims=True)
    for t in range(4):
        may = [i for i in range(E) if i not in (0, 65) and x[t, i] > -INF]
        chosen = sorted(may, key=lambda i: (-(score[t, i] + float(bias[i])), i))[:k]
        want = score[t, chosen]
        if renormalize and len(chosen):
            want = want / want.sum()
        assert ids[t].tolist() == chosen + [-1] * (k - len(chosen)), t
        # made in 64 bits and rounded once
        np.testing.assert_allclose(w[t].cpu().numpy(), list(want) + [0.0] * (k - len(chosen)),
                                   rtol=1.01 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("renormalize", [True, False])
def test_all_of_the_softmax_with_an_excluded_expert(renormalize):
    """An infinite logit under a bias of -infinity: the others' scores are 0, so they come in order
    of their biases, and weights of 0 are not divided by their sum."""
    logits = torch.tensor([[1.0, INF, 2.0, 0.5], [1.0, 2000.0, 2.0, 0.5]], device=DEV)
    bias = torch.tensor([0.0, -INF, 0.0, 0.5], device=DEV)
    w, ids = ops.route(logits, 3, bias=bias, renormalize=renormalize)
    assert ids.tolist() == [[3, 0, 2]] * 2      # (exp(-1998) is 0 in 64 bits)
    assert not w.any()


def test_routing_past_32_bits():
    """2^21 tokens of 1024 experts: the last rows start past 2^31 elements."""
    T, E, k = ops.MAX_TOKENS, 1024, 3
    logits = torch.zeros((T, E), dtype=torch.bfloat16, device=DEV)
    logits[-2, 1000], logits[-1, 500], logits[-1, 2], logits[7, 9] = 3.0, 4.0, 2.0, 1.0
    w, ids = ops.route(logits, k, id_dtype=torch.int64)
    assert ids[-2].tolist() == [1000, 0, 1] and ids[-1].tolist() == [500, 2, 0]
    assert ids[7].tolist() == [9, 0, 1]
    rest = torch.ones(T, dtype=torch.bool, device=DEV)
    rest[[-2, -1, 7]] = False
    assert (ids[rest] == torch.arange(k, device=DEV)).all()
    # a third, rounded once
    assert (w[rest] == np.float32(1 / 3)).all()
    for t, x in ((-2, [3.0, 0, 0]), (-1, [4.0, 2.0, 0]), (7, [1.0, 0, 0])):
        e = np.exp(np.array(x))
        np.testing.assert_allclose(w[t].cpu().numpy(), e / e.sum(), rtol=1.01 * 2.0 ** -24)


# ---- experts ------------------------------------------------------------------------------

BF16, F16, I8, E4 = torch.bfloat16, torch.float16, torch.int8, torch.float8_e4m3fn


def _codes(kind):
    """All 256 one-byte weights and their values; e4m3's two NaN codes are zeros here."""
    code = torch.arange(256, dtype=torch.int16).to(torch.uint8).view(torch.int8)
    if kind == E4:
        code[[0x7F, 0xFF]] = 0
        code = code.view(E4)
    return code.to(DEV), code.float().to(DEV)


def _scales(kind, rows, cols):
    return torch.ones((1, rows) if kind == I8 else (1, -(-rows // 128), -(-cols // 128)),
                      device=DEV)


@pytest.mark.parametrize("T", [1, 3, 20])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kind", [I8, E4])
def test_every_one_byte_weight(kind, dtype, T):
    """Each of the 256 codes as a weight up and as a weight down. SiLU of 64 is 64 in 32 bits and
    the routing weight 2^-6, so what goes down is the weight itself; products with one and zero
    are exact, and every value has a place in the tokens' type."""
    n = 256
    code, value = _codes(kind)
    one = torch.ones((), dtype=torch.float32).to(kind).to(DEV)
    sixty_four = torch.tensor(64.0).to(kind).to(DEV)

    def put(w, at, v):       # (one-byte floats are moved as bytes)
        w.view(torch.int8)[at] = v.view(torch.int8)

    w13 = torch.zeros((1, 2 * n, n), dtype=torch.int8, device=DEV).view(kind)
    w2 = torch.zeros((1, n, n), dtype=torch.int8, device=DEV).view(kind)
    put(w13, (0, slice(0, n), 1), sixty_four)
    put(w13, (0, slice(n, 2 * n), 0), code)
    eye = torch.arange(n, device=DEV)
    put(w2, (0, eye, eye), one)
    x = torch.zeros((T, n), dtype=dtype, device=DEV)
    x[:, :2] = 1.0
    probs = torch.full((T, 1), 2.0 ** -6, device=DEV)
    ids = torch.zeros((T, 1), dtype=torch.int32, device=DEV)
    up = ops.Experts(w13, w2, _scales(kind, 2 * n, n), _scales(kind, n, n))
    assert torch.equal(up(x, probs, ids).float(), value.expand(T, n))

    w13 = torch.zeros((1, 2 * n, n), dtype=torch.int8, device=DEV).view(kind)
    w2 = torch.zeros((1, n, n), dtype=torch.int8, device=DEV).view(kind)
    put(w13, (0, 0, 1), sixty_four)
    put(w13, (0, n, 0), one)                    # one hidden value of 1
    put(w2, (0, slice(0, n), 0), code)
    down = ops.Experts(w13, w2, _scales(kind, 2 * n, n), _scales(kind, n, n))
    assert torch.equal(down(x, probs, ids).float(), value.expand(T, n))


@pytest.mark.parametrize("T", [1, 3, 20, 300])
def test_float16_weights_and_tokens_below_its_normal_numbers(T):
    """Steps of 2^-24: not flushed, neither in experts nor in adapters. All sums are exact."""
    g = torch.Generator(device=DEV).manual_seed(T)
    tiny = torch.randint(-900, 901, (1, 16, 32), device=DEV, generator=g) * 2.0 ** -24
    w13 = torch.zeros((1, 32, 32), dtype=F16, device=DEV)
    w13[0, :16, 0] = 64.0                       # SiLU of 64
    w13[0, 16:] = tiny[0]
    w13[0, 16:, 0] = 0
    x = torch.zeros((T, 32), dtype=F16, device=DEV)
    x[:, 0] = 1.0
    x[:, 5] = 2.0 ** 10
    w2 = torch.eye(32, dtype=F16, device=DEV)[None, :, :16].contiguous()
    y = ops.Experts(w13, w2)(x, torch.full((T, 1), 2.0 ** -6, device=DEV),
                             torch.zeros((T, 1), dtype=torch.int32, device=DEV))
    assert torch.equal(y[:, :16], (tiny[0, :, 5] * 2.0 ** 10).to(F16).expand(T, 16))
    w2 = w2 * 2.0 ** -24 * 100                  # hidden values of one, small weights down
    w13[0, 16:], w13[0, 16:, 5] = 0, 1.0
    y = ops.Experts(w13, w2)(x, torch.full((T, 1), 2.0 ** -6, device=DEV),
                             torch.zeros((T, 1), dtype=torch.int32, device=DEV))
    assert torch.equal(y[:, :16], torch.full((T, 16), 100 * 2.0 ** -14, dtype=F16, device=DEV))

    a = torch.zeros((1, 8, 32), dtype=F16, device=DEV)
    a[0, :, 5] = tiny[0, :8, 5]
    b = (torch.eye(8, device=DEV)[None] * 300 * 2.0 ** -24).to(F16)
    base = torch.zeros((T, 8), dtype=F16, device=DEV)
    scale = torch.full((1,), 2.0 ** 18, device=DEV)
    y = ops.Adapters(a, b.contiguous(), scale)(x, base, torch.zeros(T, dtype=torch.int32,
                                                                    device=DEV))
    want = tiny[0, :8, 5].double() * 2.0 ** 10 * 300 * 2.0 ** -24 * 2.0 ** 18
    assert torch.equal(y, want.to(F16).expand(T, 8))


@pytest.mark.parametrize("T,k,S", [(16, 5, 3), (16, 5, 200), (9, 33, 20), (26, 5, 3), (26, 5, 200),
                                   (200, 5, 4), (31, 33, 20), (31, 33, 1100)])
def test_experts_named_twice_in_pairs_of_two_lots(T, k, S):
    """Ids are gone through 64 at a time; here tokens begin in one lot and end in the next, name
    slots twice or more, once with a weight of 0 first."""
    e = _experts(T + k, S, 64, 48, BF16)
    x, probs, ids = _tokens(T, T, k, S, 64, BF16)
    ids[:, k - 1] = ids[:, 1]
    probs[::3, 1] = 0.0
    _close(e(x, probs, ids), *_moe(e, x, probs, ids))


# ---- adapters -----------------------------------------------------------------------------

def test_adapters_of_tokens_past_32_bits():
    """2^21 tokens: rows of x, base and out that start past 2^31 elements."""
    T, H, O = ops.MAX_TOKENS, 1032, 1032
    a = torch.zeros((2, 8, H), dtype=BF16, device=DEV)
    b = torch.zeros((2, O, 8), dtype=BF16, device=DEV)
    a[1, 3, -1], b[1, -1, 3], b[1, 0, 3] = 2.0, 4.0, 1.0
    x = torch.zeros((T, H), dtype=BF16, device=DEV)
    base = torch.ones((T, O), dtype=BF16, device=DEV)
    x[-1, -1], x[-2, -1], x[5, -1] = 1.0, 3.0, 2.0
    ids = torch.full((T,), -1, dtype=torch.int32, device=DEV)
    ids[-65:], ids[5], ids[-2] = 1, 1, 0
    y = ops.Adapters(a, b)(x, base, ids)
    want = {T - 1: (3.0, 9.0), 5: (5.0, 17.0)}   # 1 + 1 * 2 * x, 1 + 4 * 2 * x
    for t, (first, last) in want.items():
        assert float(y[t, 0]) == first and float(y[t, -1]) == last
        y[t, 0] = y[t, -1] = 1.0
    assert (y == 1).all()

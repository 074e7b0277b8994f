"""The operators for many tokens (vllm_expert_cache/ops.py) on the GPU where offsets pass 32 bits:
rows, results, hidden values and weights of more than 2^32 bytes. What is far behind is compared with
the same values from a small call, which `test_gpu_many_tokens.py` has against 64 bits, or with its
formula there. Tolerances are that file's: half a step of the result's type, and 2 n 2^-24 of the sum
of the absolute values for a sum of n terms in 32 bits."""
from __future__ import annotations

import pytest
import torch

import gpu_util as gu
from vllm_expert_cache import ops

pytestmark = pytest.mark.gpu

DEV = gu.DEV
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.fixture(autouse=True)
def free_memory():
    yield
    torch.cuda.empty_cache()


def test_rows_and_back():
    T, k, S, H = 2 ** 20, 4, 64, 1032
    assert T * k * H > 2 ** 32
    g = _gen(1)
    ids = torch.randint(-1, S, (T, k), device=DEV, generator=g)
    order = ops.sort(ids, S)
    live = int(order.offsets[S])
    assert live == int((ids >= 0).sum())
    flat = ids.reshape(-1)
    pairs = order.rows[:live].long()
    key = flat[pairs]
    # by slot, and in the order of the pairs within one
    assert (key[1:] >= key[:-1]).all() and (pairs[1:] > pairs[:-1])[key[1:] == key[:-1]].all()
    assert torch.equal(order.places.reshape(-1)[pairs], torch.arange(live, device=DEV).int())
    assert (order.places.reshape(-1)[flat < 0] == -1).all() and (order.rows[live:] == -1).all()

    x = torch.randn((T, H), dtype=BF16, device=DEV, generator=g)
    rows = ops.dispatch(x, order)
    for j in range(k):
        has = (ids[:, j] >= 0).nonzero()[:, 0]
        for part in has.split(2 ** 18):
            assert torch.equal(rows[order.places[part, j].long()], x[part])
    assert not rows[live:].any()

    weights = torch.rand((T, k), device=DEV, generator=g)
    weights[::7, 1] = 0
    y = ops.combine(rows, weights, order)
    # a token's rows are copies of its own here, so its sum is its weights' times it
    of = (weights.double() * (ids >= 0)).sum(1)
    for part in (slice(0, 300), slice(T // 2, T // 2 + 300), slice(T - 300, T)):
        want = of[part, None] * x[part].double()
        bound = 2 * (k + 1) * U * want.abs()
        off = (y[part].double() - want).abs() - bound - 2.0 ** -8 * (want.abs() + bound)
        assert float(off.max()) <= 0

    dy, dw = ops.combine_grad(x, rows, weights, order)
    for part in (slice(0, 300), slice(T // 2, T // 2 + 300), slice(T - 300, T)):
        gx, at = x[part].double(), order.places[part].long()
        has = at >= 0
        want = (gx * gx).sum(1, keepdim=True) * has
        assert ((dw[part].double() - want).abs() <= 2 * (H + 1) * U * want).all()
        want = (weights[part].double().unsqueeze(2) * gx.unsqueeze(1))[has]
        got = dy[at[has]].double()
        assert ((got - want).abs() <= (2.0 ** -8 + 2 * U) * want.abs() + 2.0 ** -126).all()
    assert not dy[live:].any()


def test_rows_far_apart():
    """Three rows, each more than 2^32 bytes behind the last."""
    far = 2 ** 31 + 64
    buffer = torch.empty(2 * far + 80, dtype=BF16, device=DEV)
    x = buffer.as_strided((3, 80), (far, 1))
    x.copy_(torch.randn((3, 80), device=DEV, generator=_gen(2)))
    near = x.contiguous()
    order = ops.sort(torch.tensor([[1, 0], [0, 2], [2, 1]], device=DEV), 3)
    assert torch.equal(ops.dispatch(x, order), ops.dispatch(near, order))
    for got, want in zip(ops.quantize(x), ops.quantize(near)):
        assert torch.equal(got, want)
    w = torch.randint(-128, 128, (72, 80), dtype=I8, device=DEV, generator=_gen(3))
    lin = ops.Linear8(w, torch.rand(72, device=DEV, generator=_gen(4)))
    assert torch.equal(lin(x), lin(near))
    pairs = ops.Order(order.offsets[:3].clone(), torch.arange(3, dtype=torch.int32, device=DEV),
                      torch.arange(3, dtype=torch.int32, device=DEV).view(3, 1), 2)
    assert torch.equal(ops.combine(x, None, pairs), near)
    for got, want in zip(ops.combine_grad(x, x, torch.ones((3, 1), device=DEV), pairs),
                         ops.combine_grad(near, near, torch.ones((3, 1), device=DEV), pairs)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("O", [65552, 65549])
def test_results_of_a_projection(O):
    T, H = 66000, 96
    assert T * O > 2 ** 32
    g = _gen(5)
    w = torch.randint(-128, 128, (O, H), dtype=I8, device=DEV, generator=g)
    lin = ops.Linear8(w, torch.rand(O, device=DEV, generator=g))
    x = torch.randn((T, H), dtype=F16, device=DEV, generator=g)
    y = lin(x)
    for part in (slice(0, 70), slice(T // 2, T // 2 + 70), slice(T - 70, T)):
        assert torch.equal(y[part], lin(x[part]))


def test_hidden_values():
    T, k, S, H, I = 2 ** 18, 4, 40, 64, 4112
    assert T * k * I > 2 ** 32
    g = _gen(6)
    w13 = torch.randint(-128, 128, (S, 2 * I, H), dtype=I8, device=DEV, generator=g)
    w2 = torch.randint(-128, 128, (S, H, I), dtype=I8, device=DEV, generator=g)
    e = ops.Experts8(w13, w2, torch.rand((S, 2 * I), device=DEV, generator=g) / 400,
                     torch.rand((S, H), device=DEV, generator=g) / 400)
    x = torch.randn((T, H), dtype=BF16, device=DEV, generator=g)
    weights = torch.rand((T, k), device=DEV, generator=g)
    ids = torch.randint(-1, S, (T, k), device=DEV, generator=g)
    y = e(x, weights, ids)
    for part in (slice(0, 200), slice(T // 2, T // 2 + 200), slice(T - 200, T)):
        assert torch.equal(y[part], e(x[part], weights[part], ids[part]))


def test_weights_of_many_slots():
    T, k, S, H, I, tail = 50, 4, 1024, 2064, 1040, 24
    assert S * 2 * I * H > 2 ** 32
    g = _gen(7)
    w13 = torch.randint(-128, 128, (S, 2 * I, H), dtype=I8, device=DEV, generator=g)
    w2 = torch.randint(-128, 128, (S, H, I), dtype=I8, device=DEV, generator=g)
    s13 = torch.rand((S, 2 * I), device=DEV, generator=g) / 2000
    s2 = torch.rand((S, H), device=DEV, generator=g) / 2000
    x = torch.randn((T, H), dtype=BF16, device=DEV, generator=g)
    weights = torch.rand((T, k), device=DEV, generator=g)
    ids = torch.randint(0, tail, (T, k), dtype=torch.int32, device=DEV, generator=g)
    last = ops.Experts8(w13[-tail:], w2[-tail:], s13[-tail:], s2[-tail:])(x, weights, ids)
    assert torch.equal(ops.Experts8(w13, w2, s13, s2)(x, weights, ids + S - tail), last)

"""Pairs sorted by slot and back, and products in 8-bit integers (vllm_expert_cache/ops.py), on the
GPU against their formulas in 64 bits.

Tolerances. A result is off by half a step of its type (HALF of the value) and by what 32-bit
arithmetic leaves: one operation 2^-24 of its result, a sum of n terms at most gamma(n) = 2 n 2^-24
of the sum of their absolute values. Quantised values of 16-bit rows have to be equal: no value
that is not half way between two whole numbers is nearer to that than 2^-19 of itself. Hidden values are
computed in 32 bits, so one that lies as near to a border as its own error may be rounded to either
side: `_moe8` finds those and allows each a step.
"""
from __future__ import annotations

import ctypes

import pytest
import torch

import gpu_util as gu
from vllm_expert_cache import _lib, ops

pytestmark = pytest.mark.gpu

DEV = gu.DEV
BF16, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8
HALF = {BF16: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}
TINY = {BF16: 2.0 ** -126, F16: 2.0 ** -24, F32: 2.0 ** -126}
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, device=DEV, generator=g)


def _gamma(n):
    return 2 * n * U


def _close(got, want, bound):
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    off = ((got - want).abs() - bound)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, \
        f"off by {float((got - want).abs()[fine].max())}, {float(off.max())} over the bound"


def _ids(g, T, k, S, dtype=torch.int32, none=0.1):
    """Distinct slots a token where there are enough, some of them outside."""
    ids = torch.rand((T, max(S, k)), device=DEV, generator=g).topk(k, 1).indices % S
    drop = torch.rand((T, k), device=DEV, generator=g) < none
    outside = torch.tensor([-1, S, -2 ** 31, 2 ** 31 - 1], device=DEV)[
        torch.randint(0, 4, (T, k), device=DEV, generator=g)]
    return torch.where(drop, outside, ids).to(dtype)


def _sorted(ids, S):
    """offsets, rows and places by the definition, on the host."""
    flat = ids.reshape(-1).tolist()
    by = [[] for _ in range(S)]
    for i, e in enumerate(flat):
        if 0 <= e < S:
            by[e].append(i)
    offsets, rows, places = [0], [], [-1] * len(flat)
    for pairs in by:
        for i in pairs:
            places[i] = len(rows)
            rows.append(i)
        offsets.append(len(rows))
    rows += [-1] * (len(flat) - len(rows))
    return offsets, rows, places


# ---- sort ---------------------------------------------------------------------------------

# one pair; fewer and more pairs than a wave; one slot, most slots; both sides of one workgroup's
# pairs (4096), of the cuts by waves (64, 256, 1024) and of a lot of several workgroups'; more lots
# than workgroups
SORTS = [(1, 1, 1), (1, 8, 64), (3, 21, 5), (64, 1, 2), (65, 1, 1024), (13, 5, 7), (64, 4, 9),
         (257, 1, 64), (300, 10, 257), (128, 8, 1024), (41, 25, 1024), (512, 8, 128), (4097, 1, 128),
         (1024, 16, 128), (1025, 16, 128), (5000, 10, 910), (20000, 3, 1023), (70001, 1, 3),
         (40000, 64, 512)]


@pytest.mark.parametrize("T,k,S", SORTS)
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_sort(T, k, S, dtype):
    ids = _ids(_gen(T + k), T, k, S, dtype)
    order = ops.sort(ids, S)
    offsets, rows, places = _sorted(ids, S)
    assert order.offsets.tolist() == offsets
    assert order.rows.tolist() == rows
    assert order.places.reshape(-1).tolist() == places
    assert order.places.shape == (T, k) and order.offsets.dtype == torch.int32


def test_sort_of_one_slot_none_and_nothing():
    T, k, S = 700, 4, 12
    for e in (0, S - 1):
        order = ops.sort(torch.full((T, k), e, device=DEV), S)
        assert order.rows.tolist() == list(range(T * k))
        assert order.offsets.tolist() == [0] * (e + 1) + [T * k] * (S - e)
    for ids in (torch.full((T, k), -1, device=DEV), torch.full((T, k), S, device=DEV)):
        order = ops.sort(ids, S)
        assert order.offsets.tolist() == [0] * (S + 1)
        assert (order.rows == -1).all() and (order.places == -1).all()
    order = ops.sort(torch.empty((0, 4), dtype=torch.int32, device=DEV), 3)
    assert order.offsets.tolist() == [0] * 4 and order.rows.numel() == 0
    assert ops.dispatch(torch.empty((0, 8), device=DEV), order).shape == (0, 8)
    assert ops.combine(torch.empty((0, 8), device=DEV), None, order).shape == (0, 8)


def test_ids_of_64_bits_are_not_cut():
    ids = torch.tensor([[2 ** 32 + 1, 1], [-2 ** 32, 0]], device=DEV)
    assert ops.sort(ids, 4).places.tolist() == [[-1, 1], [-1, 0]]


def test_sort_takes_a_column_and_strided_ids():
    ids = _ids(_gen(3), 50, 4, 9)
    assert torch.equal(ops.sort(ids[:, 0], 9).places, ops.sort(ids[:, :1].contiguous(), 9).places)
    assert torch.equal(ops.sort(ids[:, ::2], 9).rows, ops.sort(ids[:, ::2].contiguous(), 9).rows)
    assert torch.equal(ops.sort(ids.t(), 9).rows, ops.sort(ids.t().contiguous(), 9).rows)


# ---- dispatch and combine -----------------------------------------------------------------

# rows of one value, below, at and past a wave's 1 KB and 4 KB, of odd length; below, at and past a
# piece of 16 bytes; past the caches, whole and with tails
MOVES = [(12, 3, 5, 3), (12, 3, 5, 4), (12, 3, 5, 8), (12, 3, 5, 9), (40, 8, 17, 500),
         (3, 2, 4, 12296), (2100, 8, 16, 4104), (1, 1, 1, 1), (1, 8, 64, 2048), (5, 3, 4, 7), (37, 10, 19, 1045), (16, 2, 3, 512),
         (9, 4, 300, 513), (130, 6, 31, 2056), (3, 64, 1024, 4100), (700, 2, 8, 48)]


def _case(seed, T, k, S, H, dtype, none=0.1):
    g = _gen(seed)
    ids = _ids(g, T, k, S, none=none)
    order = ops.sort(ids, S)
    live = int(order.offsets[-1])
    return g, order, live, order.rows[:live].long()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,k,S,H", MOVES)
def test_dispatch(T, k, S, H, dtype):
    g, order, live, pair = _case(T * k + H, T, k, S, H, dtype)
    x = _randn(g, T, H).to(dtype)
    rows = ops.dispatch(x, order)
    assert torch.equal(rows[:live], x[pair // k])
    assert not rows[live:].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,k,S,H", MOVES)
def test_combine(T, k, S, H, dtype):
    g, order, live, pair = _case(T * k + H, T, k, S, H, dtype)
    y = _randn(g, T * k, H).to(dtype)
    y[live:] = float("nan")  # rows of no pair are not read
    w = torch.softmax(_randn(g, T, k), 1)
    for weights in (w, None):
        f = torch.ones_like(w).double() if weights is None else w.double()
        terms = y[:live].double() * f.view(-1, 1)[pair]
        zero = torch.zeros((T, H), dtype=torch.float64, device=DEV)
        want = zero.index_add(0, pair // k, terms)
        size = zero.index_add(0, pair // k, terms.abs())
        got = ops.combine(y, weights, order)
        assert got.dtype == dtype
        _close(got, want, _gamma(k) * size + HALF[dtype] * (want.abs() + _gamma(k) * size)
               + TINY[dtype])


def _grads(out, inputs, grad):
    return torch.autograd.grad(out, inputs, grad)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("T,k,S,H", MOVES)
def test_gradients(T, k, S, H, dtype):
    g, order, live, pair = _case(T * k + H, T, k, S, H, dtype)
    x = _randn(g, T, H).to(dtype).requires_grad_()
    gr = _randn(g, T * k, H).to(dtype)
    gr[live:] = float("nan")
    dx, = _grads(ops.dispatch(x, order), x, gr)
    zero = torch.zeros((T, H), dtype=torch.float64, device=DEV)
    want = zero.index_add(0, pair // k, gr[:live].double())
    size = zero.index_add(0, pair // k, gr[:live].double().abs())
    _close(dx, want, _gamma(k) * size + HALF[dtype] * (want.abs() + _gamma(k) * size)
           + TINY[dtype])

    y = _randn(g, T * k, H).to(dtype)
    y[live:] = float("nan")
    y.requires_grad_()
    w = torch.softmax(_randn(g, T, k), 1).requires_grad_()
    go = _randn(g, T, H).to(dtype)
    dy, dw = _grads(ops.combine(y, w, order), (y, w), go)
    want_y = torch.zeros((T * k, H), dtype=torch.float64, device=DEV)
    want_y[:live] = go.double()[pair // k] * w.detach().double().view(-1, 1)[pair]
    _close(dy, want_y, (U + HALF[dtype]) * 1.01 * want_y.abs() + TINY[dtype])
    assert not dy[live:].any()
    terms = go.double()[pair // k] * y.detach()[:live].double()
    want_w = torch.zeros(T * k, dtype=torch.float64, device=DEV)
    size_w = want_w.clone()
    want_w[pair], size_w[pair] = terms.sum(1), terms.abs().sum(1)
    _close(dw.reshape(-1), want_w, _gamma(H) * size_w + U * want_w.abs())

    # one of the two alone, and without autograd, bit for bit
    alone, = _grads(ops.combine(y, w.detach(), order), y, go)
    assert torch.equal(alone, dy)
    alone, = _grads(ops.combine(y.detach(), w, order), w, go)
    assert torch.equal(alone, dw)
    with torch.no_grad():
        dy2, dw2 = ops.combine_grad(go, y, w, order)
        assert torch.equal(dy2, dy) and torch.equal(dw2, dw)
        assert torch.equal(ops.combine(gr, None, order), dx)


def test_gradients_against_differences():
    """f = <combine(dispatch(x) * v, w), c> is linear in each of x, v and w, so its difference over
    any step is its derivative's: in float32, values of about one, sums of n terms."""
    T, k, S, H = 11, 3, 5, 37
    g, order, live, pair = _case(5, T, k, S, H, F32)
    x = _randn(g, T, H).requires_grad_()
    v = _randn(g, T * k, H).requires_grad_()
    w = _randn(g, T, k).requires_grad_()
    c = _randn(g, T, H)

    def f(x, v, w):
        return (ops.combine(ops.dispatch(x, order) * v, w, order).double() * c.double()).sum()

    grads = _grads(f(x, v, w), (x, v, w), torch.ones((), dtype=torch.float64, device=DEV))
    args = [x.detach(), v.detach(), w.detach()]
    for i, d in enumerate(grads):
        step = torch.randn(d.shape, device=DEV, generator=g)
        # of every term: two products' roundings, the sum's of k, the result's; of a gradient the
        # same, with a sum of H in the weights'
        a = [v.abs().double() for v in args]
        a[i] += step.abs().double()
        size = float((a[0][pair // k] * a[1][:live] * a[2].view(-1, 1)[pair]
                      * c.double().abs()[pair // k]).sum())
        with torch.no_grad():
            up, down = list(args), list(args)
            up[i], down[i] = args[i] + step, args[i] - step
            diff = float(f(*up) - f(*down)) / 2
            want = float((d.double() * (up[i].double() - down[i].double()) / 2).sum())
        assert abs(diff - want) <= 3 * (_gamma(H) + _gamma(k) + 4 * U) * size, (i, diff, want)


def test_differentiable_once():
    order = ops.sort(_ids(_gen(2), 5, 2, 3), 3)
    x = torch.ones((5, 8), device=DEV, requires_grad=True)
    y = torch.ones((10, 8), device=DEV, requires_grad=True)
    for out, leaf in ((ops.dispatch(x, order), x), (ops.combine(y, None, order), y)):
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(out.sum(), leaf, create_graph=True)


def test_a_weight_of_zero_hides_infinities():
    order = ops.sort(torch.tensor([[0, 1], [1, 0]], device=DEV), 2)
    y = torch.ones((4, 8), device=DEV)
    y[order.places[0, 1]] = float("inf")
    y[order.places[1, 0]] = float("nan")
    w = torch.tensor([[0.5, 0.0], [0.0, 2.0]], device=DEV)
    out = ops.combine(y, w, order)
    assert (out[0] == 0.5).all() and (out[1] == 2.0).all()
    assert not torch.isfinite(ops.combine(y, None, order)).any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_of_other_strides(dtype):
    T, k, S, H = 21, 4, 6, 77
    g, order, live, pair = _case(9, T, k, S, H, dtype)
    wide = _randn(g, T, 2 * H + 5).to(dtype)
    for x in (wide[:, 3:3 + H], wide[:, :2 * H:2], wide[:, 1].unsqueeze(1).expand(T, H),
              wide[0, :H].expand(T, H), wide.t()[:T, :T]):
        assert torch.equal(ops.dispatch(x, order), ops.dispatch(x.contiguous(), order))
    rows = _randn(g, T * k, 2 * H + 5).to(dtype)
    w = torch.rand((k, T), device=DEV, generator=g).t()
    for y in (rows[:, 3:3 + H], rows[:, :2 * H:2], rows[0, :H].expand(T * k, H)):
        got = ops.combine(y, w, order)
        assert torch.equal(got, ops.combine(y.contiguous(), w.contiguous(), order))
    # a gradient that is one value everywhere, as a sum's is
    x = wide[:, 3:3 + H].detach().requires_grad_()
    ops.dispatch(x, order).sum().backward()
    count = torch.zeros(T, device=DEV).index_add(0, pair // k, torch.ones(live, device=DEV))
    assert torch.equal(x.grad.float(), count.unsqueeze(1).expand(T, H))


def test_shared_inputs_add_their_gradients():
    """Weights that all tokens share, and one tensor as tokens of two orders."""
    T, k, S, H = 12, 3, 4, 16
    g, order, live, pair = _case(10, T, k, S, H, F32, none=0.0)
    w = torch.rand(k, device=DEV, generator=g).requires_grad_()
    x = _randn(g, T, H).requires_grad_()
    out = ops.combine(ops.dispatch(x, order), w.expand(T, k), order)
    dx, dw = _grads(out, (x, w), torch.ones_like(out))
    total = w.detach().double().sum()
    _close(dx, total.expand(T, H), 8 * U * total.expand(T, H))
    want = x.detach().double().sum().expand(k)
    _close(dw, want, (_gamma(T * H) * x.detach().double().abs().sum()).expand(k))


def test_dispatch_captured():
    T, k, S, H = 40, 4, 16, 96
    g = _gen(12)
    ids, x, gr = _ids(g, T, k, S), _randn(g, T, H).to(BF16), _randn(g, T, H).to(BF16)
    w = torch.rand((T, k), device=DEV, generator=g)

    def step():
        order = ops.sort(ids, S)
        rows = ops.dispatch(x, order)
        dy, dw = ops.combine_grad(gr, rows, w, order)
        return (order.offsets, order.rows, rows, ops.combine(rows, w, order), dy, dw,
                ops.combine(dy, None, order))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        ids.copy_(_ids(g, T, k, S))
        x.copy_(_randn(g, T, H))
        w.copy_(torch.rand((T, k), device=DEV, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(out, step()):
            assert torch.equal(got, want)


def test_recording_is_refused_in_a_capture():
    T, k, S, H = 4, 2, 3, 16
    order = ops.sort(_ids(_gen(1), T, k, S), S)
    x = torch.ones((T, H), device=DEV, requires_grad=True)
    y = torch.ones((T * k, H), device=DEV, requires_grad=True)
    alive = ops.dispatch(x, order), ops.combine(y, None, order)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError, match="captured"):
            ops.dispatch(x, order)
        with pytest.raises(ValueError, match="captured"):
            ops.combine(y, None, order)
        with torch.no_grad():
            out = ops.dispatch(x, order)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.dispatch(x.detach(), order))
    alive[0].sum().backward()
    assert x.grad.shape == (T, H)


def test_on_another_stream():
    T, k, S, H = 300, 6, 40, 1000
    g = _gen(13)
    ids, x = _ids(g, T, k, S), _randn(g, T, H).to(BF16).requires_grad_()
    order = ops.sort(ids, S)
    want = ops.dispatch(x, order)
    dwant, = _grads(want, x, want.detach())
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        order2 = ops.sort(ids, S)
        got = ops.dispatch(x, order2)
        dgot, = _grads(got, x, got.detach())
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(dgot, dwant)


def test_rows_behind_the_result_stay():
    """C entry points with wider rows: nothing but the rows' values is written."""
    import ctypes
    T, k, S, H = 7, 3, 5, 33
    g, order, live, pair = _case(14, T, k, S, H, F32)
    x = _randn(g, T, H)
    lib, P = gu.lib(), ctypes.c_void_p
    wide = torch.full((T * k + 1, H + 7), 5.0, device=DEV)
    assert lib.expert_cache_dispatch(gu.ptr(x), 0, H, gu.ptr(order.places), gu.ptr(order.rows), T,
                                     k, H, gu.ptr(wide), H + 7, gu.stream()) == 0
    torch.cuda.synchronize()
    assert (wide[:, H:] == 5).all() and (wide[T * k] == 5).all()
    assert torch.equal(wide[:T * k, :H], ops.dispatch(x, order))
    back = torch.full((T + 1, H + 3), 5.0, device=DEV)
    assert lib.expert_cache_combine(gu.ptr(wide), 0, H + 7, P(None), gu.ptr(order.places), T, k, H,
                                    gu.ptr(back), H + 3, gu.stream()) == 0
    torch.cuda.synchronize()
    assert (back[:, H:] == 5).all() and (back[T] == 5).all()
    assert torch.equal(back[:T, :H], ops.combine(ops.dispatch(x, order), None, order))


# ---- 8-bit integers -----------------------------------------------------------------------

def _quantized(x):
    """(whole numbers, scales) by the formula in 64 bits."""
    x = x.double()
    m = x.abs().amax(1)
    live = m >= 2.0 ** -119
    q = torch.where(live.unsqueeze(1), 127 * x / torch.where(live, m, 1.0).unsqueeze(1), 0.0)
    return q.round(), torch.where(live, m, 0.0)


def _hard_rows(g, T, H, dtype):
    """Random rows, rows of halves of the largest, tiny, huge, constant and zero rows."""
    x = _randn(g, T, H)
    kind = torch.arange(T, device=DEV) % 7
    steps = torch.randint(-254, 255, (T, H), device=DEV, generator=g).float()
    x = torch.where((kind == 1).unsqueeze(1), steps / 254 * 1.5, x)     # multiples of half a step
    x = torch.where((kind == 2).unsqueeze(1), x * 2.0 ** -14, x)
    x = torch.where((kind == 3).unsqueeze(1), (x * 8000).clamp(-65504, 65504), x)
    x = torch.where((kind == 4).unsqueeze(1), torch.full_like(x, -0.37), x)
    x = torch.where((kind == 5).unsqueeze(1), torch.zeros_like(x), x)
    x = x.to(dtype)
    half = x.abs().amax(1, keepdim=True).float() / 2
    return torch.where((kind == 6).unsqueeze(1) & (x.float() > 0), half.to(dtype).expand(T, H), x)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,H", [(1, 1), (7, 16), (15, 1045), (29, 2048), (8, 8192), (8, 8200),
                                 (9, 14336), (3, 40009), (600, 129), (1025, 129), (1026, 2049),
                                 (1030, 4096), (1024, 4097)])
def test_quantize(T, H, dtype):
    x = _hard_rows(_gen(T + H), T, H, dtype)
    q, scales = ops.quantize(x)
    want, m = _quantized(x)
    assert q.dtype == I8 and q.shape == (T, H) and torch.equal(q.double(), want)
    # the quotient in 64 bits, rounded once (a tensor divided by a number is multiplied by 1 / 127)
    assert torch.equal(scales, (m / torch.full_like(m, 127)).float())
    if H % 16:  # the rest of the last 16 bytes
        rest = q.as_strided((T, -H % 16), (q.stride(0), 1), H)
        assert not rest.any()


def test_quantize_extremes():
    x = torch.zeros((6, 40), dtype=BF16, device=DEV)
    x[0, 3] = 2.0 ** -120
    x[1, 3] = 2.0 ** -119
    x[2, 5], x[2, 6] = float("inf"), 1
    x[3, 39] = float("nan")
    x[4, 0], x[4, 1] = -3.0e38, 1.5e38
    x[5, 1] = -float("inf")
    q, s = ops.quantize(x)
    assert not q[0].any() and s[0] == 0
    assert q[1, 3] == 127 and s[1] == 2.0 ** -119 / 127
    assert q[4, 0] == -127 and q[4, 1] in (63, 64) and torch.isfinite(s[4])
    for row in (2, 3, 5):
        assert torch.isnan(s[row]) and not q[row].any()


def _whole(g, *shape):
    return (_randn(g, *shape) * 40).round().clamp(-128, 127).to(I8)


# one value; lengths below, at and past a step of 128 and with tails; outputs and tokens below, at
# and past a tile; every size of tile
LINEARS = [(1, 1, 1), (1, 16, 16), (2, 128, 128), (3, 129, 17), (5, 1045, 1003), (16, 2048, 96),
           (17, 144, 130), (31, 400, 128), (33, 256, 257), (64, 272, 64), (65, 1024, 48),
           (128, 128, 128), (129, 640, 384), (200, 96, 1000), (256, 512, 256), (257, 16, 513),
           (300, 4112, 520), (513, 1040, 1045),
           # few tokens quantised beside the product, as many values as that takes and one row more
           (3, 4096, 24), (3, 5000, 24), (2, 8192, 20), (7, 2304, 18), (4, 4096, 40), (8, 2048, 33), (9, 2048, 33), (1, 16384, 20), (1, 16400, 20), (48, 1000, 50),
           # cut along the length: 6, 3 and 8 parts, of which the last is short or empty
           (70, 6200, 130), (130, 6160, 1029), (20, 8300, 77),
           # tiles of 128 and 256: filled, ragged, odd outputs, one step and several
           (1000, 160, 2344), (1100, 96, 2043), (2500, 144, 2568), (2437, 272, 2701), (2304, 128, 2816)]


def _linear(q, m, lin, bias):
    """(result, bound without the last rounding) from whole numbers and the rows' maxima."""
    y = q @ lin.w[:, :lin.H].double().t()
    y = y * (m / 127).unsqueeze(1) * lin.scale.double().view(1, -1)
    b = bias.double().unsqueeze(0) if bias is not None else torch.zeros_like(y)
    # the scale's own rounding, the sum's to 32 bits, two products, the bias's sum
    return y + b, 1.01 * U * (4 * y.abs() + (y + b).abs())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T,H,O", LINEARS)
def test_linear8(T, H, O, dtype):
    g = _gen(T + H + O)
    bias = _randn(g, O) if O % 2 else None
    w = _whole(g, O, H)
    lin = ops.Linear8(w, (0.5 + torch.rand(O, device=DEV, generator=g)) * H ** -0.5 / 40, bias)
    assert (lin.w.data_ptr() == w.data_ptr()) == (H % 16 == 0)
    x = _randn(g, T, H).to(dtype)
    want, bound = _linear(*_quantized(x), lin, bias)
    for out in (dtype, F32):
        y = lin(x, dtype=out)
        assert y.dtype == out
        _close(y, want, bound + HALF[out] * (want.abs() + bound) + TINY[out])
    # the same from a call of quantize, and repeated, bit for bit
    q, scales = ops.quantize(x)
    assert torch.equal(lin(q, scales, dtype=dtype), lin(x))
    assert torch.equal(lin(x), lin(x))


def test_linear8_extreme_sums():
    """Every product -128 * -128 or -127 * 128, as long as sums may be."""
    H = ops.MAX_LENGTH8
    w = torch.full((3, H), -128, dtype=I8, device=DEV)
    w[1] = 127
    lin = ops.Linear8(w, torch.ones(3, device=DEV))
    q = torch.full((2, H), -128, dtype=I8, device=DEV)
    q[1] = 127
    y = lin(q, torch.ones(2, device=DEV), dtype=F32)
    want = q.double() @ w.double().t()
    assert torch.equal(y, want.float())


def test_linear8_of_other_strides():
    g = _gen(21)
    T, H, O = 40, 176, 72
    lin = ops.Linear8(_whole(g, O, H), torch.rand(O, device=DEV, generator=g))
    wide = _randn(g, T, 2 * H + 9).to(BF16)
    for x in (wide[:, 5:5 + H], wide[:, :2 * H:2], wide[0, :H].expand(T, H)):
        assert torch.equal(lin(x), lin(x.contiguous()))
    s = torch.rand(2 * T, device=DEV, generator=g)
    q = _whole(g, T, 2 * H + 16)
    for x in (q[:, :H], q[:, 1:1 + H], q[:, :2 * H:2], q[:, H + 16:]):
        assert torch.equal(lin(x, s[::2]), lin(x.contiguous(), s[::2].contiguous()))
    # weights that lie otherwise are copied, whole rows of a wider matrix are used as they lie
    for w in (_whole(g, H, O).t(), _whole(g, O, H + 3)[:, 3:], _whole(g, O, H + 16)[:, 16:]):
        a, b = ops.Linear8(w, lin.scale), ops.Linear8(w.contiguous(), lin.scale)
        assert torch.equal(a(wide[:, :H]), b(wide[:, :H]))
    # rows of the result apart
    out = torch.full((T, O + 5), 7.0, dtype=BF16, device=DEV)
    lin(wide[:, :H], out=out[:, 2:2 + O])
    assert torch.equal(out[:, 2:2 + O], lin(wide[:, :H]))
    assert (out[:, :2] == 7).all() and (out[:, 2 + O:] == 7).all()


# One row has no stride: in tiles (O from 8192 on) the rows that a tile has behind it touch nothing,
# whatever stride is given. Long rows are cut along the length, with scales that end where they end.
@pytest.mark.parametrize("H,O", [(1001, 8201), (6211, 8191 + 2), (70, 8192)])
@pytest.mark.parametrize("dtype", [BF16, I8])
def test_linear8_of_one_row_of_any_stride(H, O, dtype):
    g = _gen(23)
    w = _whole(g, O, H)
    lin = ops.Linear8(w, torch.rand(O, device=DEV, generator=g))
    x, s = ops.quantize(_randn(g, 1, H).to(BF16))
    if dtype == BF16:
        x, s = _randn(g, 1, H).to(BF16), None
        q, m = _quantized(x)
        want, bound = _linear(q, m, lin, None)
    else:
        want = x.double() @ w.double().t() * s.double() * lin.scale.double()
        bound = _gamma(3) * want.abs()
    kind = 1 if dtype == BF16 else 3
    h, size = _lib.lib(), ctypes.c_long()
    assert h.expert_cache_linear8_workspace(lin._at, kind, 1, ctypes.addressof(size)) == 0
    work = torch.empty(max(size.value, 16), dtype=torch.uint8, device=DEV)
    for x_stride, out_stride in ((0, 0), (16, 4), (x.stride(0), O), (2 ** 22, 2 ** 20)):
        out = torch.full((O + 64,), 7.0, device=DEV)
        torch.cuda.synchronize()
        assert h.expert_cache_linear8(lin._at, x.data_ptr(), kind, x_stride,
                                      None if s is None else s.data_ptr(), 1, out.data_ptr(), 0,
                                      out_stride, work.data_ptr(), None) == 0
        torch.cuda.synchronize()
        _close(out[None, :O], want, bound)
        assert (out[O:] == 7).all()


def test_linear8_shows_infinities_in_their_rows_alone():
    g = _gen(22)
    lin = ops.Linear8(_whole(g, 50, 96), torch.rand(50, device=DEV, generator=g))
    x = _randn(g, 70, 96).to(F16)
    want = lin(x)
    x[3, 7], x[69, 0] = float("inf"), float("nan")
    got = lin(x)
    rows = torch.ones(70, dtype=torch.bool, device=DEV)
    rows[[3, 69]] = False
    assert torch.equal(got[rows], want[rows]) and torch.isnan(got[~rows]).all()


def test_no_tokens():
    lin = ops.Linear8(torch.ones((8, 16), dtype=I8, device=DEV), torch.ones(8, device=DEV))
    assert lin(torch.empty((0, 16), dtype=BF16, device=DEV)).shape == (0, 8)
    assert ops.quantize(torch.empty((0, 16), dtype=BF16, device=DEV))[0].shape == (0, 16)


# ---- experts8 -----------------------------------------------------------------------------

def _experts(seed, S, H, I):
    g = _gen(seed)
    def slab(rows, cols):
        return _whole(g, S, rows, cols), \
            (0.5 + torch.rand((S, rows), device=DEV, generator=g)) * cols ** -0.5 / 40
    w13, s13 = slab(2 * I, H)
    w2, s2 = slab(H, I)
    return ops.Experts8(w13, w2, s13, s2)


def _moe8(e, x, probs, ids):
    """(output, bound on its error) by the formula in 64 bits."""
    T, H = x.shape
    I = e.I
    q, m = _quantized(x)
    scale = m / 127
    y = torch.zeros((T, H), dtype=torch.float64, device=DEV)
    err, size = torch.zeros_like(y), torch.zeros_like(y)
    for s in set(ids.reshape(-1).tolist()):
        if not 0 <= s < e.S:
            continue
        t, j = torch.nonzero((ids == s) & (probs != 0), as_tuple=True)
        if not len(t):
            continue
        gu_ = (q[t] @ e.w13[s].double().t()) * e.w13_scale[s].double() * scale[t, None]
        g, u = gu_[:, :I], gu_[:, I:]
        h = g * torch.sigmoid(g) * u
        # g and u are off by 4 U of themselves, which silu makes (1 + |g|) times as much; the
        # exponential by (2 |g| + 4) U, quotient and products by U each
        dh = h.abs() * U * (4 * (1 + g.abs()) + 4 + 2 * g.abs() + 4 + 4)
        m2 = h.abs().amax(1, keepdim=True)
        d2 = (dh / m2.clamp(min=1e-300)).amax(1, keepdim=True)  # of the row's maximum, at most
        v = 127 * h / m2.clamp(min=1e-300)
        dv = 127 * dh / m2.clamp(min=1e-300) + v.abs() * (d2 + 4 * U)
        q2 = v.round()
        step = ((v - v.floor() - 0.5).abs() <= dv).double()  # may be rounded to either side
        w2 = e.w2[s].double() * e.w2_scale[s].double().unsqueeze(1)
        out = (q2 @ w2.t()) * (m2 / 127)
        off = (step @ w2.abs().t()) * (m2 / 127) + out.abs() * (d2 + 5 * U)
        p = probs[t, j].double().unsqueeze(1)
        y.index_add_(0, t, p * out)
        err.index_add_(0, t, p.abs() * off)
        size.index_add_(0, t, p.abs() * (out.abs() + off))
    err = err + _gamma(ids.shape[1]) * size
    return y, err * 1.01 + HALF[x.dtype] * (y.abs() + err) + TINY[x.dtype]


# one pair; tails of H and I; more and fewer pairs than slots; slots of no, few and many pairs,
# below, at and past a tile's rows; more than one tile along every side
LAYERS = [(1, 1, 1, 16, 16), (1, 2, 4, 128, 128), (2, 4, 6, 272, 144), (5, 3, 3, 400, 48),
          (16, 8, 20, 144, 272), (33, 1, 1, 160, 80), (40, 5, 37, 64, 32), (129, 2, 2, 256, 192),
          (300, 4, 9, 528, 208), (513, 8, 16, 96, 112), (700, 3, 1024, 48, 16), (64, 64, 70, 32, 64)]


def _tokens(seed, T, k, S, H, dtype, id_dtype):
    g = _gen(seed + 1)
    x = _randn(g, T, H).to(dtype)
    probs = torch.softmax(_randn(g, T, k), 1)
    probs[torch.rand((T, k), device=DEV, generator=g) < 0.05] = 0
    return x, probs, _ids(g, T, k, S, id_dtype, none=0.05 if T > 1 else 0)


@pytest.mark.parametrize("dtype,id_dtype", [(BF16, torch.int32), (F16, torch.int64)])
@pytest.mark.parametrize("T,k,S,H,I", LAYERS)
def test_experts8(T, k, S, H, I, dtype, id_dtype):
    e = _experts(T + k, S, H, I)
    x, probs, ids = _tokens(T + S, T, k, S, H, dtype, id_dtype)
    got = e(x, probs, ids)
    want, bound = _moe8(e, x, probs, ids)
    _close(got, want, bound)
    assert torch.equal(got, e(x, probs, ids))
    # a token's result does not depend on the tokens beside it
    some = torch.arange(0, T, max(1, T // 5), device=DEV)
    assert torch.equal(e(x[some], probs[some], ids[some]), got[some])


FILLS = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128, 129, 159, 161, 191, 193, 223,
         225, 255, 256, 257]


@pytest.mark.parametrize("fills", [FILLS[:8] + [0] * 20, FILLS, [256 + n for n in FILLS]], ids=len)
def test_experts8_of_every_fill(fills):
    """Slots of as many pairs as fill a tile, its rounds and their operands, and one more or less;
    tiles of 32, 128 and 256 rows. The rows of a slot's neighbours stay its neighbours'."""
    S, H, I = len(fills), 144, 80
    e = _experts(60 + S, S, H, I)
    g = _gen(sum(fills))
    ids = torch.repeat_interleave(torch.arange(S, device=DEV), torch.tensor(fills, device=DEV))
    ids = ids[torch.randperm(len(ids), device=DEV, generator=g)].unsqueeze(1)
    x = _randn(g, len(ids), H).to(BF16)
    probs = torch.rand((len(ids), 1), device=DEV, generator=g) + 0.1
    got = e(x, probs, ids)
    _close(got, *_moe8(e, x, probs, ids))
    assert torch.equal(got, e(x, probs, ids))


def test_experts8_of_one_slot_and_of_none():
    e = _experts(3, 8, 128, 64)
    x, probs, ids = _tokens(4, 300, 2, 8, 128, BF16, torch.int32)
    assert not e(x, probs, torch.full_like(ids, -1)).any()
    assert not e(x, torch.zeros_like(probs), ids).any()
    for slot in (0, 7):
        same = torch.full_like(ids, slot)  # the same slot twice a token
        _close(e(x, probs, same), *_moe8(e, x, probs, same))
    assert e(x[:0], probs[:0], ids[:0]).shape == (0, 128)


def test_experts8_shows_infinities_in_their_tokens_alone():
    e = _experts(5, 6, 96, 48)
    x, probs, ids = _tokens(6, 90, 3, 6, 96, BF16, torch.int32)
    ids, probs = ids.clamp(0, 5), probs + 0.01
    want = e(x, probs, ids)
    x[4, 9], x[88, 0] = float("inf"), float("nan")
    got = e(x, probs, ids)
    rows = torch.ones(90, dtype=torch.bool, device=DEV)
    rows[[4, 88]] = False
    assert torch.equal(got[rows], want[rows]) and torch.isnan(got[~rows]).all()


def test_experts8_into_wider_rows_and_from_them():
    T, k, S, H = 50, 4, 10, 112
    e = _experts(7, S, H, 32)
    x, probs, ids = _tokens(8, T, k, S, H, F16, torch.int64)
    want = e(x, probs, ids)
    wide = torch.full((T, H + 11), 3.0, dtype=F16, device=DEV)
    e(x, probs, ids, out=wide[:, 1:1 + H])
    assert torch.equal(wide[:, 1:1 + H], want)
    assert (wide[:, 0] == 3).all() and (wide[:, 1 + H:] == 3).all()
    apart = torch.zeros((T, 2 * H + 1), dtype=F16, device=DEV)
    apart[:, 1:1 + H] = x
    assert torch.equal(e(apart[:, 1:1 + H], probs.t().contiguous().t(), ids), want)


def test_experts8_captured_on_two_streams_at_once():
    """Two captured calls of one handle, replayed beside each other, with eager work between."""
    T, k, S, H, I = 200, 4, 12, 160, 96
    e = _experts(9, S, H, I)
    lin = ops.Linear8(_whole(_gen(30), 64, H), torch.rand(64, device=DEV))
    sets = [list(_tokens(10 + i, T, k, S, H, BF16, torch.int32)) for i in range(2)]
    e(*sets[0]), lin(sets[0][0])
    graphs, outs = [], []
    for s in sets:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = e(*s)
            outs.append((y, lin(y)))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in sets]
    for i in range(4):
        for j, s in enumerate(sets):
            for old, new in zip(s, _tokens(50 + 2 * i + j, T, k, S, H, BF16, torch.int32)):
                old.copy_(new)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for s, (y, z) in zip(sets, outs):
            assert torch.equal(y, e(*s)) and torch.equal(z, lin(y))


def test_a_layer_of_the_parts():
    """Routing, sorting, products slot by slot and back, and a projection behind: what Experts8
    does as one call, by the parts, as a training program would put them together."""
    T, k, S, H, I = 96, 4, 8, 128, 64
    g = _gen(40)
    e = _experts(11, S, H, I)
    logits, x = _randn(g, T, S), _randn(g, T, H).to(BF16)
    weights, ids = ops.route(logits, k)
    got = e(x, weights, ids)
    order = ops.sort(ids, S)
    q, scales = ops.quantize(ops.dispatch(x, order))
    rows = torch.zeros((T * k, H), device=DEV)
    at = order.offsets.tolist()
    for s in range(S):
        part = slice(at[s], at[s + 1])
        up = ops.Linear8(e.w13[s], e.w13_scale[s])(q[part], scales[part], dtype=F32).double()
        h = torch.nn.functional.silu(up[:, :I]) * up[:, I:]
        hq, m = _quantized(h)
        down = ops.Linear8(e.w2[s], e.w2_scale[s])
        rows[part] = down(hq.to(I8), (m / 127).float(), dtype=F32)
    by_parts = ops.combine(rows, weights, order)
    want, bound = _moe8(e, x, weights, ids)
    _close(got, want, bound)
    _close(by_parts.double(), want, bound)  # the same formula in parts, rounded less

"""Performance cases of the operators for many tokens: pairs of token and slot sorted by slot and
back, with gradients, and products in 8-bit integers.

Operators (`op`):

  dispatch  pairs of token and slot in the slots' order, and the tokens' rows in that order; with
            `grad` the gradient of the tokens.
  combine   rows in the slots' order back to their tokens, weighted and summed; with `grad` the
            gradients of the rows and of the weights.
  linear8   a projection in 8-bit integers: every token quantised with a scale of its own, weights
            with a scale a channel; with `split` quantised by a call of its own, as projections
            that share their tokens do it.
  experts8  a whole mixture-of-experts layer in 8-bit integers for any number of tokens, over
            experts in slots: both projections' inputs quantised row by row.

Sizes are those of the package's workloads (experts of 2048 x 768 in int8 with a scale a row,
of 4096 x 14336, of 7168 x 2048) or generic.
"""
from __future__ import annotations

import math
import os
import sys
from types import SimpleNamespace

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _package():
    pkg = os.path.join(os.getcwd(), "vllm-expert-cache_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from vllm_expert_cache import ops

    return ops


def _sorted(name, op, tokens, top_k, slots, hidden, type="bf16", grad=False, pad=0, id64=False,
            zipf=0.4):
    return {"name": name, "op": op, "tokens": tokens, "top_k": top_k, "slots": slots,
            "hidden": hidden, "type": type, "grad": grad, "pad": pad, "id64": id64, "zipf": zipf}


def _linear8(name, tokens, hidden, out, type="bf16", bias=False, split=False, gap=0):
    return {"name": name, "op": "linear8", "tokens": tokens, "hidden": hidden, "out": out,
            "type": type, "bias": bias, "split": split, "gap": gap}


def _experts8(name, tokens, top_k, slots, hidden, inter, type="bf16", pad=0, id64=False, zipf=0.4):
    return {"name": name, "op": "experts8", "tokens": tokens, "top_k": top_k, "slots": slots,
            "hidden": hidden, "inter": inter, "type": type, "pad": pad, "id64": id64, "zipf": zipf}


def listed():
    return [
        # one token's rows for its eight experts: latency alone
        _sorted("dispatch-1", "dispatch", 1, 8, 64, 2048),
        # a ragged float32 training batch of odd rows, 21 of them padding
        _sorted("dispatch-517-odd-grad", "dispatch", 517, 3, 48, 1001, type="f32", grad=True,
                pad=21, id64=True),
        # a training step's chunk on 128 experts
        _sorted("dispatch-4096-grad", "dispatch", 4096, 8, 128, 2048, grad=True),
        # one token's expert outputs summed up
        _sorted("combine-1", "combine", 1, 8, 64, 2048),
        # a decode batch of 300 in float16 with rows of odd length
        _sorted("combine-300-f16-odd", "combine", 300, 10, 257, 1045, type="f16", zipf=1.0),
        # a training step's chunk on 128 experts
        _sorted("combine-8192-grad", "combine", 8192, 8, 128, 2048, grad=True),
        # a projection of single-user decode
        _linear8("linear8-1", 1, 2048, 4096),
        # projections that share their tokens: 37 rows of odd lengths out of a wider buffer
        _linear8("linear8-37-odd-split", 37, 1045, 1003, type="f16", bias=True, split=True, gap=19),
        # a prefill chunk through a large projection
        _linear8("linear8-4096", 4096, 4096, 14336),
        # a decode batch of 33 users, two rows of padding, on small experts
        _experts8("experts8-33", 33, 8, 64, 2048, 768, pad=2, zipf=0.8),
        # a prefill chunk on 128 small experts
        _experts8("experts8-2048", 2048, 8, 128, 2048, 768),
        # a prefill chunk on eight large experts
        _experts8("experts8-2048-large", 2048, 2, 8, 4096, 14336, id64=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    op = rng.choice(["dispatch", "combine", "linear8", "experts8"])
    if op in ("dispatch", "combine"):
        slots, hidden = _log(rng, 4, 512), _log(rng, 16, 7168)
        if rng.random() < 0.6:
            hidden = -(-hidden // 8) * 8
        top_k = rng.randint(1, min(10, slots))
        type = rng.choice(["f32", "bf16", "bf16", "f16"])
        size = 4 if type == "f32" else 2
        tokens = max(1, min(_log(rng, 1, 8192), int(2.7e8) // (top_k * hidden * size)))
        return _sorted("", op, tokens, top_k, slots, hidden, type, grad=rng.random() < 0.6,
                       pad=rng.choice([0, 0, rng.randint(1, 40)]), id64=rng.random() < 0.3,
                       zipf=round(rng.uniform(0.0, 1.3), 2))
    if op == "linear8":
        hidden, out = _log(rng, 16, 14336), _log(rng, 16, 16384)
        if rng.random() < 0.6:
            hidden, out = -(-hidden // 16) * 16, -(-out // 16) * 16
        tokens = max(1, min(_log(rng, 1, 8192), int(2.4e11) // (hidden * out),
                            int(1.2e8) // max(hidden, out)))
        return _linear8("", tokens, hidden, out, type=rng.choice(["bf16", "bf16", "f16"]),
                        bias=rng.random() < 0.4, split=rng.random() < 0.4,
                        gap=rng.choice([0, 0, rng.randint(1, 64)]))
    hidden, inter = 16 * _log(rng, 16, 448), 16 * _log(rng, 4, 512)
    slots = max(4, min(_log(rng, 4, 300), int(1.4e9) // (3 * hidden * inter)))
    top_k = rng.randint(1, min(10, slots // 2))
    tokens = max(1, min(_log(rng, 1, 8192), int(2.4e11) // (top_k * hidden * inter),
                        int(1.3e8) // (top_k * max(hidden, inter))))
    return _experts8("", tokens, top_k, slots, hidden, inter,
                     type=rng.choice(["bf16", "bf16", "f16"]),
                     pad=rng.choice([0, 0, rng.randint(1, 40)]), id64=rng.random() < 0.3,
                     zipf=round(rng.uniform(0.0, 1.0), 2))


# ---- inputs ------------------------------------------------------------------------------

def _randn(gen, *shape):
    return torch.randn(shape, device=DEV, generator=gen)


def _int8(gen, *shape, std):
    """Weights of standard deviation `std` in 8 bits, and a scale for every row."""
    w = torch.empty(shape, dtype=torch.int8, device=DEV)
    for part in (w.split(1) if w.dim() == 3 else (w,)):
        part.copy_((_randn(gen, *part.shape) * 36).round_().clamp_(-127, 127))
    return w, (0.5 + torch.rand(shape[:-1], device=DEV, generator=gen)) * (std / 36)


def _routes(gen, case):
    """k slots a token by popularity, shuffled over the slots, and their weights; padded rows
    have none."""
    T, pad, S, k = (case[f] for f in ("tokens", "pad", "slots", "top_k"))
    rank = torch.randperm(S, device=DEV, generator=gen) + 1.0
    u = torch.rand((T + pad, S), device=DEV, generator=gen).clamp_(1e-6, 1 - 1e-6)
    ids = (-case["zipf"] * rank.log() - (-u.log()).log()).topk(k, dim=1).indices
    probs = torch.softmax(_randn(gen, T + pad, k), dim=1)
    ids[T:] = -1
    probs[T:] = 0.0
    return ids.to(torch.int64 if case["id64"] else torch.int32), probs


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = SimpleNamespace(case=case, handle=None, order=None, grad=None)
    dtype = TYPES[case["type"]]
    if case["op"] == "linear8":
        T, H, O = case["tokens"], case["hidden"], case["out"]
        s.x = _randn(gen, T, H + case["gap"]).to(dtype)[:, :H]
        s.w, s.scale = _int8(gen, O, H, std=H ** -0.5)
        s.bias = 0.1 * _randn(gen, O) if case["bias"] else None
        if own:
            s.handle = _package().Linear8(s.w, s.scale, s.bias)
        return s
    s.ids, s.probs = _routes(gen, case)
    rows, H = case["tokens"] + case["pad"], case["hidden"]
    if case["op"] == "experts8":
        S, I = case["slots"], case["inter"]
        s.x = _randn(gen, rows, H).to(dtype)
        s.w13, s.s13 = _int8(gen, S, 2 * I, H, std=H ** -0.5)
        s.w2, s.s2 = _int8(gen, S, H, I, std=I ** -0.5)
        if own:
            s.handle = _package().Experts8(s.w13, s.w2, s.s13, s.s2)
        return s
    pairs = rows * case["top_k"]
    if case["op"] == "dispatch":
        s.x = _randn(gen, rows, H).to(dtype).requires_grad_(case["grad"])
        if case["grad"]:
            s.grad = _randn(gen, pairs, H).to(dtype)
        return s
    s.y = _randn(gen, pairs, H).to(dtype).requires_grad_(case["grad"])
    s.probs.requires_grad_(case["grad"])
    if case["grad"]:
        s.grad = _randn(gen, rows, H).to(dtype)
    s.order = _package().sort(s.ids, case["slots"]) if own else _plain_sort(s.ids, case["slots"])
    return s


# ---- one pass ----------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    with torch.no_grad():
        return {"dispatch": _plain_dispatch, "combine": _plain_combine, "linear8": _plain_linear8,
                "experts8": _plain_experts8}[s.case["op"]](s)


def _own(s):
    ops, c = _package(), s.case
    if c["op"] == "dispatch":
        order = ops.sort(s.ids, c["slots"])
        rows = ops.dispatch(s.x, order)
        out = [order.offsets, order.rows, order.places, rows]
        return out + list(torch.autograd.grad(rows, s.x, s.grad)) if c["grad"] else out
    if c["op"] == "combine":
        out = ops.combine(s.y, s.probs, s.order)
        return [out, *torch.autograd.grad(out, (s.y, s.probs), s.grad)] if c["grad"] else [out]
    if c["op"] == "linear8":
        if not c["split"]:
            return [s.handle(s.x)]
        q, scales = ops.quantize(s.x)
        return [s.handle(q, scales, dtype=s.x.dtype), scales]
    return [s.handle(s.x, s.probs, s.ids)]


def _plain_sort(ids, S):
    """The pairs of every slot side by side in their own order: where each slot begins, the pair
    at every place (-1 behind the last) and the place of every pair (-1: none)."""
    flat = ids.reshape(-1).long()
    n = flat.numel()
    key = torch.where((flat >= 0) & (flat < S), flat, S)
    by, at = key.sort(stable=True)
    offsets = torch.searchsorted(by, torch.arange(S + 1, device=ids.device))
    live = torch.arange(n, device=ids.device) < offsets[S]
    places = torch.empty_like(flat)
    places[at] = torch.where(live, torch.arange(n, device=ids.device), -1)
    return SimpleNamespace(offsets=offsets.int(), rows=torch.where(live, at, -1).int(),
                           places=places.view(ids.shape).int())


def _plain_sum(rows, places):
    """For every token the 32-bit sum of the rows at its places."""
    picked = rows.float()[places.clamp(min=0).long()]
    return torch.where((places >= 0).unsqueeze(2), picked, 0.0).sum(1)


def _plain_dispatch(s):
    order = _plain_sort(s.ids, s.case["slots"])
    live = (order.rows >= 0).unsqueeze(1)
    rows = torch.where(live, s.x[(order.rows.clamp(min=0) // s.ids.shape[1]).long()], 0.0)
    out = [order.offsets, order.rows, order.places, rows.to(s.x.dtype)]
    if s.grad is not None:
        out.append(_plain_sum(s.grad, order.places).to(s.x.dtype))
    return out


def _plain_combine(s):
    places, k = s.order.places, s.case["top_k"]
    at = places.clamp(min=0).long()
    used = (places >= 0) & (s.probs != 0)
    picked = s.y[at].float()
    out = torch.where(used.unsqueeze(2), picked * s.probs.unsqueeze(2), 0.0).sum(1).to(s.y.dtype)
    if s.grad is None:
        return [out]
    g = s.grad.float()
    pair = s.order.rows.clamp(min=0).long()
    dy = s.probs.reshape(-1)[pair].unsqueeze(1) * g[pair // k]
    dy = torch.where((s.order.rows >= 0).unsqueeze(1), dy, 0.0).to(s.y.dtype)
    dp = torch.where(places >= 0, (picked * g.unsqueeze(1)).sum(2), 0.0)
    return [out, dy, dp]


def _plain_quantize(x):
    """Rows as whole numbers up to 127, and what 1 stands for. The numbers in 64 bits: 16-bit
    values are often half way between two (half of the largest one is 63.5)."""
    most = x.float().abs().amax(1, keepdim=True)
    live = most >= 2.0 ** -119
    q = torch.where(live, x.double() * 127.0 / torch.where(live, most, 1.0), 0.0).round()
    return q.float(), torch.where(live, most, 0.0).squeeze(1) / 127.0


def _plain_linear8(s):
    q, scales = _plain_quantize(s.x)
    y = (q @ s.w.float().T) * scales.unsqueeze(1) * s.scale
    if s.bias is not None:
        y = y + s.bias
    return [y.to(s.x.dtype), scales] if s.case["split"] else [y.to(s.x.dtype)]


def _plain_experts8(s):
    """Pairs in the slots' order, every slot's in blocks of its own, so that one batched product
    takes all blocks."""
    T, H = s.x.shape
    k, S, I = s.case["top_k"], s.case["slots"], s.case["inter"]
    order = _plain_sort(torch.where(s.probs != 0, s.ids.long(), -1), S)
    rows = 16
    while rows < 256 and rows * S < T * k:
        rows *= 2
    count = order.offsets.diff().long()
    ends = ((count + rows - 1) // rows).cumsum(0)
    blocks = T * k // rows + S  # at most
    slot = torch.searchsorted(ends, torch.arange(blocks, device=DEV), right=True).clamp(max=S - 1)
    live = order.rows >= 0
    pair = torch.where(live, order.rows, 0).long()
    of = s.ids.reshape(-1)[pair].long().clamp(0, S - 1)
    first = (ends - (count + rows - 1) // rows) * rows
    place = torch.arange(T * k, device=DEV) - order.offsets.long()[of] + first[of]
    place = torch.where(live, place, blocks * rows)  # the last row takes what belongs to none
    q, scales = _plain_quantize(s.x)

    def product(a, w, scale, row_scale):
        laid = a.new_zeros((blocks * rows + 1, a.shape[1]))
        laid[place] = a
        laid = laid[:-1].view(blocks, rows, -1).transpose(1, 2).contiguous()
        y = torch.bmm(w[slot].float(), laid).transpose(1, 2) * scale[slot].unsqueeze(1)
        y = torch.cat([y.reshape(blocks * rows, -1), y.new_zeros((1, w.shape[1]))])
        return y[place] * row_scale.unsqueeze(1)

    token = pair // k
    g, u = product(q[token], s.w13, s.s13, scales[token]).chunk(2, 1)
    q2, scales2 = _plain_quantize(g / (1 + (-g).exp()) * u)
    y = product(q2, s.w2, s.s2, scales2) * s.probs.reshape(-1)[pair].unsqueeze(1)
    return [_plain_sum(y, order.places).to(s.x.dtype)]


# ---- from the definition, in 64 bits -----------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"dispatch": _exact_dispatch, "combine": _exact_combine, "linear8": _exact_linear8,
                "experts8": _exact_experts8}[case["op"]](case, s)


def _exact_lists(ids, S):
    """The pairs of every slot, slot by slot."""
    flat = ids.reshape(-1).cpu().numpy().astype(np.int64)
    named = np.flatnonzero((flat >= 0) & (flat < S))
    return flat, named[np.argsort(flat[named], kind="stable")]


def _exact_dispatch(c, s):
    flat, at = _exact_lists(s.ids, c["slots"])
    token = torch.from_numpy(at // c["top_k"]).to(DEV)
    rows = torch.zeros((len(flat), c["hidden"]), dtype=torch.float64, device=DEV)
    rows[:len(at)] = s.x.detach().double()[token]
    out = [None, None, None, rows]
    if s.grad is not None:
        dx = torch.zeros(s.x.shape, dtype=torch.float64, device=DEV)
        out.append(dx.index_add_(0, token, s.grad[:len(at)].double()))
    return out


def _exact_combine(c, s):
    flat, at = _exact_lists(s.ids, c["slots"])
    k, H, T = c["top_k"], c["hidden"], s.ids.shape[0]
    pair = torch.from_numpy(at).to(DEV)
    p = s.probs.detach().double().reshape(-1)
    y = s.y.detach()[:len(at)].double()
    out = torch.zeros((T, H), dtype=torch.float64, device=DEV)
    out.index_add_(0, pair // k, y * p[pair].unsqueeze(1))
    if s.grad is None:
        return [out]
    g = s.grad.double()[pair // k]
    dy = torch.zeros((len(flat), H), dtype=torch.float64, device=DEV)
    dy[:len(at)] = g * p[pair].unsqueeze(1)
    dp = torch.zeros(len(flat), dtype=torch.float64, device=DEV)
    dp[pair] = (g * y).sum(1)
    return [out, dy, dp.view(T, k)]


def _exact_quantize(x):
    x = x.double()
    largest = x.abs().max(1).values
    divisor = largest.where(largest > 0, torch.ones_like(largest)).unsqueeze(1)
    return (127 * x / divisor).round(), largest / 127


def _exact_linear8(c, s):
    q, scale = _exact_quantize(s.x)
    y = torch.empty((c["tokens"], c["out"]), dtype=torch.float64, device=DEV)
    for first in range(0, c["out"], 2048):
        of = slice(first, first + 2048)
        y[:, of] = q @ s.w[of].double().t() * torch.outer(scale, s.scale[of].double())
        if s.bias is not None:
            y[:, of] += s.bias[of].double()
    return [y, scale] if c["split"] else [y]


def _exact_experts8(c, s):
    I = c["inter"]
    q, scale = _exact_quantize(s.x)
    out = torch.zeros(s.x.shape, dtype=torch.float64, device=DEV)
    ids, probs = s.ids.cpu(), s.probs.cpu().double()
    for slot in range(c["slots"]):
        t, j = torch.nonzero((ids == slot) & (probs != 0), as_tuple=True)
        if not len(t):
            continue
        rows = t.to(DEV)
        gu = (q[rows] @ s.w13[slot].double().t()) * s.s13[slot].double() * scale[rows, None]
        h, hs = _exact_quantize(gu[:, :I] * torch.sigmoid(gu[:, :I]) * gu[:, I:])
        y = (h @ s.w2[slot].double().t()) * s.s2[slot].double() * hs[:, None]
        out.index_add_(0, rows, y * probs[t, j].to(DEV)[:, None])
    return [out]


# ---- what a pass cannot do without -------------------------------------------------------

def work(case):
    """Inputs read once and outputs written once; of the slots, those that the step's ids name
    (as many as that many draws by popularity meet)."""
    T = case["tokens"]
    if case["op"] == "linear8":
        H, O = case["hidden"], case["out"]
        return {"bytes": 2.0 * T * (H + O) + O * H + 4.0 * O * (2 if case["bias"] else 1)
                + (4.0 * T if case["split"] else 0.0), "flops": 2.0 * T * H * O}
    H, k, S = case["hidden"], case["top_k"], case["slots"]
    rows, id_bytes = T + case["pad"], 8 if case["id64"] else 4
    pairs = rows * k
    if case["op"] == "experts8":
        I = case["inter"]
        p = np.arange(1, S + 1, dtype=np.float64) ** -case["zipf"]
        lo, hi = 0.0, 1e6  # the weight at which a token meets k slots on average
        for _ in range(60):
            mid = (lo + hi) / 2
            lo, hi = (mid, hi) if (1 - np.exp(-mid * p)).sum() < k else (lo, mid)
        met = float((1 - np.exp(-lo * p * T)).sum())
        return {"bytes": met * (3 * H * I + 4 * (2 * I + H)) + 4.0 * rows * H
                + pairs * (4 + id_bytes), "flops": 6.0 * T * k * H * I}
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "dispatch":
        moved = size * H * (T + pairs) + 8.0 * pairs + 4.0 * (S + 1) + pairs * id_bytes
        if case["grad"]:
            moved += size * H * (T * k + rows)
        return {"bytes": float(moved), "flops": float(T * k * H if case["grad"] else 0)}
    moved = size * H * (T * k + rows) + 8.0 * pairs
    if case["grad"]:
        moved += size * H * (T + pairs) + 4.0 * pairs
    return {"bytes": float(moved), "flops": 2.0 * T * k * H * (3 if case["grad"] else 1)}

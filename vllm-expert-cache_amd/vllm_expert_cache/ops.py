"""Operators around the slot cache: the routing that makes its ids, and the products over what
its slots hold.

    weights, ids = route(logits, top_k)               # expert ids from the gate's logits
    slots = cache.refresh(ids)                        # experts into slots (cache.py)
    y = Experts(w13_slots, w2_slots)(x, weights, slots)

    slots = adapter_cache.refresh(adapter_ids)        # the same for adapters of requests
    y = Adapters(a_slots, b_slots)(x, projected, slots)

For many tokens, in parts or as a whole layer in 8-bit integers:

    order = sort(slots, S)                            # pairs of token and slot, slot by slot
    rows = dispatch(x, order)                         # every slot's tokens side by side
    y = combine(products_of(rows, order.offsets), weights, order)
    y = Experts8(w13_slots, w2_slots, s13, s2)(x, weights, slots)
    y = Linear8(w, w_scale)(x)                        # a projection; quantize(x) is its first half

`Experts`, `Adapters`, `Linear8` and `Experts8` check their weights once and are kept like the
weights themselves; a cache's slot tensors never move, so a handle over them stays good. Weights are
used as they lie, without another layout (but see `Linear8`). Calls run on the current stream of the
tensors' device, allocate only their result and a workspace through torch, and read nothing back, so
they can be captured.

`dispatch` and `combine` have a backward pass. The others have none: with gradients enabled, a tensor
that requires one (a handle's weights: when the handle is made) is refused. None has a forward-mode
derivative: a tensor with a tangent (torch.autograd.forward_ad) is refused everywhere. They are no
registered torch operators, and a call that torch.jit.trace or make_fx would record is refused.

ValueError names an argument that an operator does not take; nothing has run then.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib

_TOKENS = {torch.bfloat16: 1, torch.float16: 2}
_LOGITS = {torch.float32: 0, **_TOKENS}
_BYTES = {torch.int8: 3, torch.float8_e4m3fn: 4}
_SCORING = {"softmax": 0, "sigmoid": 1}
_ID_BYTES = {torch.int32: 4, torch.int64: 8}
_BLOCK = 128  # rows and columns of e4m3 weights that share a scale

MAX_PAIRS = 1024    # tokens x top_k of one Experts call
MAX_TOP_K = 64
MAX_EXPERTS = 1024  # of one routing
MAX_GROUPS = 64
MAX_RANK = 256
MAX_TOKENS = 1 << 21   # of one routing or Adapters call
MAX_OUTPUTS = 1 << 21  # of an adapter
MAX_LENGTH = 1 << 24   # of a row of weights: H and I
MAX_SORTED = 1 << 24   # pairs of one sort: tokens x top_k
MAX_ROW = 1 << 20      # values of a row that is dispatched, combined or quantised
MAX_MOVED = 1 << 35    # bytes of the tokens' rows that are dispatched or combined
MAX_TOKENS8 = 1 << 23  # rows that are quantised: tokens of 8-bit products, Experts8's pairs
MAX_LENGTH8 = 131056   # of a sum of 8-bit products, which 32 bits hold
MAX_BYTES8 = 7 << 28   # of Experts8's quantised tokens, and of an expert's w13
MAX_VALUES8 = 1 << 36  # of its hidden values, and of its pairs' outputs
MAX_RESULTS8 = 1 << 38 # of a Linear8


def _check(rc: int, name: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{name} failed rc={rc}")


# The current stream's handle without building a torch.cuda.Stream around it (a microsecond of
# each call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


# Whether torch.jit.trace runs, and whether a graph of torch's own operators is recorded from real
# tensors (make_fx). Neither sees a kernel launch, only the result's allocation.
_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)
_mode = getattr(torch._C, "_get_dispatch_mode", lambda key: None)
_PROXY = getattr(getattr(torch._C, "_TorchDispatchModeKey", None), "PROXY", None)


def _on_device(device: torch.device, call, *args):
    """call(*args, stream) on the current stream of `device`, with that device current."""
    if _tracing() or _mode(_PROXY) is not None:
        raise ValueError("a trace would keep the result's memory without what fills it: leave the "
                         "call outside what is traced")
    index = device.index
    if index == torch.cuda.current_device():
        return call(*args, _raw_stream(index))
    with torch.cuda.device(device):
        return call(*args, _raw_stream(index))


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` as rows that the kernels can load 16 bytes at a time: itself, or a copy."""
    n, step = t.shape[0], t.stride()
    if step[1] != 1 or t.data_ptr() % 16 or (n > 1 and (step[0] % 8 or step[0] < t.shape[1])):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _ids(ids: torch.Tensor, device) -> tuple[torch.Tensor, int]:
    nbytes = _ID_BYTES.get(ids.dtype)
    if nbytes is None or ids.device != device:
        raise ValueError(f"ids must be int32 or int64 on {device}, not {ids.dtype} on {ids.device}")
    return ids if ids.is_contiguous() else ids.contiguous(), nbytes


def _on_gpu(*tensors) -> torch.device:
    device = tensors[0].device
    if device.type != "cuda":
        raise ValueError(f"tensors must be on a GPU, not on {device}")
    for t in tensors[1:]:
        if t is not None and t.device != device:
            raise ValueError(f"tensors are on {device} and on {t.device}")
    return device


def _no_gradient(*tensors) -> None:
    """Refuses a call that autograd would have to record."""
    for t in tensors:
        if t is not None and t.requires_grad:
            raise ValueError(f"a tensor {list(t.shape)} requires a gradient and there is no backward "
                             f"pass: detach it, or call under torch.no_grad()")


def _no_tangent(*tensors) -> None:
    """Refuses a tensor with a forward-mode derivative: the kernels would drop it, and the result
    count as a constant. Only inside a level of `torch.autograd.forward_ad` has a tensor one, so calls
    look for a level first; whether gradients are enabled makes no difference to it."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f"a tensor {list(t.shape)} has a forward-mode derivative and there is "
                             f"none of the result: pass forward_ad.unpack_dual(t).primal")


def _graded(*weights) -> list:
    """A handle's weights that require a gradient: looked for once, since each look at a tensor
    is a tenth of a microsecond of a call."""
    return [w for w in weights if w is not None and w.requires_grad]


def route(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax",
          bias: torch.Tensor | None = None, groups: int = 1, topk_groups: int = 1,
          renormalize: bool = True, scale: float = 1.0,
          id_dtype: torch.dtype = torch.int32) -> tuple[torch.Tensor, torch.Tensor]:
    """The `top_k` experts of every token: (weights float32 [T, top_k], ids [T, top_k]).

    logits  [T, E] float32, bfloat16 or float16; E up to 1024
    scoring "softmax" of a row, or "sigmoid" of each logit
    bias    float32 [E] added to the scores for the selection alone
    groups  select from the best `topk_groups` of this many equal groups (up to 64). A group
            counts as its best expert, with a bias as the sum of its two best.
    renormalize  divide the selected scores by their sum
    scale   factor on the weights

    Among equals the lowest id comes first. Experts whose logit or bias is NaN or -inf are never
    selected (one that a bias excludes still counts in the softmax); where too few are left the
    id is -1 and the weight 0. Selected scores that are all 0 give weights of 0."""
    kind = _LOGITS.get(logits.dtype)
    if kind is None or logits.dim() != 2:
        raise ValueError(f"logits must be float32, bfloat16 or float16 [T, E], not {logits.dtype} "
                         f"{list(logits.shape)}")
    code, nbytes = _SCORING.get(scoring), _ID_BYTES.get(id_dtype)
    if code is None or nbytes is None:
        raise ValueError(f"scoring {scoring!r} (softmax or sigmoid), ids of {id_dtype} (int32 or "
                         f"int64)")
    T, E = logits.shape
    if T > MAX_TOKENS:
        raise ValueError(f"{T} tokens (at most {MAX_TOKENS})")
    if not 0 < E <= MAX_EXPERTS:
        raise ValueError(f"{E} experts (1 to {MAX_EXPERTS})")
    if not 1 <= groups <= MAX_GROUPS or E % groups or not 1 <= topk_groups <= groups:
        raise ValueError(f"{topk_groups} of {groups} groups of {E} experts (at most {MAX_GROUPS} "
                         f"equal groups)")
    if not 1 <= top_k <= min(MAX_TOP_K, topk_groups * (E // groups)):
        raise ValueError(f"top_k {top_k} of {topk_groups} x {E // groups} experts (at most "
                         f"{MAX_TOP_K})")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (E,) or
                             not bias.is_contiguous()):
        raise ValueError(f"bias must be contiguous float32 [{E}], not {bias.dtype} "
                         f"{list(bias.shape)}")
    device = _on_gpu(logits, bias)
    if forward_ad._current_level >= 0:
        _no_tangent(logits, bias)
    if torch.is_grad_enabled() and (logits.requires_grad or bias is not None):
        _no_gradient(logits, bias)
    step = logits.stride()
    if step[1] != 1 or step[0] < E:
        logits, step = logits.contiguous(), (E, 1)
    weights = logits.new_empty((T, top_k), dtype=torch.float32)
    ids = logits.new_empty((T, top_k), dtype=id_dtype)
    _check(_on_device(device, _lib.lib().expert_cache_route, logits.data_ptr(), kind, step[0],
                      None if bias is None else bias.data_ptr(), T, E, top_k, code, groups,
                      topk_groups, 1 if renormalize else 0, scale, weights.data_ptr(),
                      ids.data_ptr(), nbytes), "expert_cache_route")
    return weights, ids


def _need(ok, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _scales(s, shape, name: str, device):
    _need(s is not None and s.dtype == torch.float32 and s.is_contiguous() and
          s.data_ptr() % 16 == 0, f"{name} must be contiguous, 16-byte aligned float32")
    _need(tuple(s.shape) == shape or tuple(s.shape) == shape + (1,),
          f"{name} must be {list(shape)}, not {list(s.shape)}")
    _need(s.device == device, f"{name} is on {s.device}, not {device}")


class Experts:
    """The experts of one layer, in slots or all of them: a whole MoE layer for a few tokens.

    w13  [S, 2*I, H]: gate rows, then up rows        w2  [S, H, I]
    in bfloat16 or float16 (the tokens' type); int8 with float32 scales a row, w13_scale
    [S, 2*I] or [S, 2*I, 1] and w2_scale [S, H] or [S, H, 1]; or float8_e4m3fn with float32
    scales a 128 x 128 block, [S, ceil(2*I/128), ceil(H/128)] and [S, ceil(H/128), ceil(I/128)].
    H and I are multiples of 8, with one-byte weights of 16.

    Activations are not quantised: one-byte weights are widened to the tokens' type and sums are
    32-bit. Hidden values are rounded to two bfloat16 (2^-17 of the value), the result to its type.
    The same call gives the same bits; a token's last bits may differ with the tokens beside it.
    Infinite hidden values or weights of w2 make infinities or NaN of the outputs they reach."""

    def __init__(self, w13: torch.Tensor, w2: torch.Tensor, w13_scale: torch.Tensor | None = None,
                 w2_scale: torch.Tensor | None = None):
        _need(w13.dim() == 3 and w2.dim() == 3 and w13.dtype == w2.dtype,
              "w13 and w2 must be [S, 2*I, H] and [S, H, I] of one type")
        S, two, H = w13.shape
        _need(two % 2 == 0 and tuple(w2.shape) == (S, H, two // 2) and min(S, two, H) > 0,
              f"w13 {list(w13.shape)} does not go with w2 {list(w2.shape)}")
        dtype = w13.dtype
        _need(dtype in _TOKENS or dtype in _BYTES, f"weights of {dtype} are not supported")
        least = 16 if dtype in _BYTES else 8
        _need(H % least == 0 and (two // 2) % least == 0,
              f"H {H} and I {two // 2} must be multiples of {least}")
        _need(max(H, two // 2) <= MAX_LENGTH, f"H {H} and I {two // 2} (at most {MAX_LENGTH})")
        for name, w in (("w13", w13), ("w2", w2)):
            _need(w.is_contiguous() and w.data_ptr() % 16 == 0,
                  f"{name} must be contiguous and 16-byte aligned")
        device = _on_gpu(w13, w2)
        if dtype == torch.int8:
            _scales(w13_scale, (S, two), "w13_scale", device)
            _scales(w2_scale, (S, H), "w2_scale", device)
        elif dtype == torch.float8_e4m3fn:
            _scales(w13_scale, (S, -(-two // _BLOCK), -(-H // _BLOCK)), "w13_scale", device)
            _scales(w2_scale, (S, -(-H // _BLOCK), -(-two // 2 // _BLOCK)), "w2_scale", device)
        else:
            _need(w13_scale is None and w2_scale is None, f"weights of {dtype} have no scales")
        self.w13, self.w2, self.w13_scale, self.w2_scale = w13, w2, w13_scale, w2_scale
        self.S, self.H, self.I, self.device = S, H, two // 2, device
        self.dtypes = (dtype,) if dtype in _TOKENS else tuple(_TOKENS)
        self._structs = {}
        for t in self.dtypes:
            e = _lib.Experts(S, H, two // 2, _TOKENS[t], _BYTES.get(dtype, _TOKENS[t]),
                             w13.data_ptr(), w2.data_ptr(),
                             *[s.data_ptr() if s is not None else None
                               for s in (w13_scale, w2_scale)])
            self._structs[t] = (e, ctypes.addressof(e))
        self._graded = _graded(w13, w2, w13_scale, w2_scale)
        self._bytes: dict = {}

    def __call__(self, x: torch.Tensor, topk_weights: torch.Tensor, slot_ids: torch.Tensor,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        """The layer's output [T, H] for tokens x [T, H]: the sum over their slots of the routing
        weight (float32 [T, top_k]) times the expert. slot_ids [T, top_k] are int32 or int64;
        T x top_k is at most 1024. A pair whose id is outside [0, S) or whose weight is 0 adds
        nothing (and an infinity in that expert does not show); a token without any other
        pair gets zeros. `out`, if given, has contiguous rows and overlaps no other argument."""
        struct = self._structs.get(x.dtype)
        if struct is None or x.dim() != 2 or x.shape[1] != self.H or x.device != self.device:
            raise ValueError(f"x must be [T, {self.H}] on {self.device} of {self.dtypes}, not "
                             f"{list(x.shape)} on {x.device} of {x.dtype}")
        T, shape = x.shape[0], slot_ids.shape
        if len(shape) != 2 or shape[0] != T or topk_weights.shape != shape or \
                topk_weights.dtype != torch.float32 or topk_weights.device != self.device:
            raise ValueError(f"slot_ids {list(shape)} and float32 topk_weights must be [{T}, top_k] "
                             f"on {self.device}, not {topk_weights.dtype} "
                             f"{list(topk_weights.shape)} on {topk_weights.device}")
        k = shape[1]
        if not 1 <= k <= MAX_TOP_K or T * k > MAX_PAIRS:
            raise ValueError(f"{T} tokens x top_k {k} (top_k at most {MAX_TOP_K}, {MAX_PAIRS} in "
                             f"all)")
        if forward_ad._current_level >= 0:
            _no_tangent(x, topk_weights, out, self.w13, self.w2, self.w13_scale, self.w2_scale)
        if torch.is_grad_enabled() and (x.requires_grad or topk_weights.requires_grad or
                                        self._graded or out is not None):
            _no_gradient(x, topk_weights, out, *self._graded)
        ids, nbytes = _ids(slot_ids, self.device)
        if not topk_weights.is_contiguous():
            topk_weights = topk_weights.contiguous()
        x = _rows(x)
        given = out is not None
        if not given:
            out = x.new_empty((T, self.H))
        else:
            _out(out, x.dtype, (T, self.H), self.device)
        h, at = _lib.lib(), struct[1]
        size = self._bytes.get((T, k))
        if size is None:
            size = self._bytes[T, k] = _workspace(h.expert_cache_moe_workspace, at, T, k)
        work = x.new_empty(size, dtype=torch.uint8)
        _check(_on_device(self.device, h.expert_cache_moe, at, x.data_ptr(), x.stride(0),
                          topk_weights.data_ptr(), ids.data_ptr(), nbytes, T, k, out.data_ptr(),
                          out.stride(0), work.data_ptr()), "expert_cache_moe")
        if given:
            _written(out)
        return out


def _workspace(entry, struct, *sizes) -> int:
    size = ctypes.c_long()
    _check(entry(struct, *sizes, ctypes.addressof(size)), entry.__name__)
    return max(16, size.value)


def _out(out, dtype, shape, device) -> None:
    _need(out.dtype == dtype and tuple(out.shape) == shape and out.device == device and
          out.stride(1) == 1 and (shape[0] < 2 or out.stride(0) >= shape[1]),
          f"out must be {dtype} {list(shape)} on {device} with contiguous rows")


def _written(out) -> None:
    """Counts the write into a caller's `out`, as torch does for its own operators: a backward pass
    that saved what it held is refused then, and doesn't go on with what it holds now."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


class Adapters:
    """Low-rank adapters in slots, added for every token to a projection that all share.

    a  [S, R, H], b  [S, O, R] in bfloat16 or float16; scales float32 [S] or None (1).
    H and R are multiples of 8, R at most 256. Sums are 32-bit; between the products a token's
    values are rounded to two bfloat16, with what `Experts` says of those."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor | None = None):
        _need(a.dim() == 3 and b.dim() == 3 and a.dtype == b.dtype and a.dtype in _TOKENS,
              "a and b must be [S, R, H] and [S, O, R] in bfloat16 or float16")
        S, R, H = a.shape
        _need(b.shape[0] == S and b.shape[2] == R and min(*a.shape, *b.shape) > 0,
              f"a {list(a.shape)} does not go with b {list(b.shape)}")
        _need(H % 8 == 0 and R % 8 == 0 and R <= MAX_RANK,
              f"H {H} and R {R} must be multiples of 8, R at most {MAX_RANK}")
        _need(H <= MAX_LENGTH and b.shape[1] <= MAX_OUTPUTS,
              f"H {H} (at most {MAX_LENGTH}) and {b.shape[1]} outputs (at most {MAX_OUTPUTS})")
        for name, w in (("a", a), ("b", b)):
            _need(w.is_contiguous() and w.data_ptr() % 16 == 0,
                  f"{name} must be contiguous and 16-byte aligned")
        self.device = _on_gpu(a, b, scales)
        if scales is not None:
            _scales(scales, (S,), "scales", self.device)
        self.a, self.b, self.scales = a, b, scales
        self.S, self.R, self.H, self.O, self.dtype = S, R, H, b.shape[1], a.dtype
        self._struct = _lib.Adapters(S, H, b.shape[1], R, _TOKENS[a.dtype], a.data_ptr(),
                                     b.data_ptr(), scales.data_ptr() if scales is not None
                                     else None)
        self._at = ctypes.addressof(self._struct)
        self._graded = _graded(a, b, scales)
        self._bytes: dict = {}

    def __call__(self, x: torch.Tensor, base: torch.Tensor, slot_ids: torch.Tensor,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        """base + scale * b[s] (a[s] x) for every token, s its slot id ([T], int32 or int64);
        x [T, H], base [T, O]. A token whose id is outside [0, S) has no adapter: its row is
        base's. `out` may be base, whose rows without an adapter are then not written; any
        other `out` overlaps no other argument."""
        dtype, device = self.dtype, self.device
        if x.dim() != 2 or x.shape[1] != self.H or x.dtype != dtype or x.device != device:
            raise ValueError(f"x must be {dtype} [T, {self.H}] on {device}, not {x.dtype} "
                             f"{list(x.shape)} on {x.device}")
        T = x.shape[0]
        if base.shape != (T, self.O) or base.dtype != dtype or base.device != device:
            raise ValueError(f"base must be {dtype} [{T}, {self.O}] on {device}, not {base.dtype} "
                             f"{list(base.shape)} on {base.device}")
        if slot_ids.shape != (T,) or T > MAX_TOKENS:
            raise ValueError(f"slot_ids must be [{T}], not {list(slot_ids.shape)}, of at most "
                             f"{MAX_TOKENS} tokens")
        if forward_ad._current_level >= 0:
            _no_tangent(x, base, out, self.a, self.b, self.scales)
        if torch.is_grad_enabled() and (x.requires_grad or base.requires_grad or self._graded or
                                        out is not None):
            _no_gradient(x, base, out, *self._graded)
        ids, nbytes = _ids(slot_ids, device)
        x = _rows(x)
        given = out is not None
        if not given:
            out = x.new_empty((T, self.O))
        else:
            _out(out, dtype, (T, self.O), device)
        if base.stride(1) != 1 or (T > 1 and base.stride(0) < self.O):
            base = base.contiguous()
        h = _lib.lib()
        size = self._bytes.get(T)
        if size is None:
            size = self._bytes[T] = _workspace(h.expert_cache_adapt_workspace, self._at, T)
        work = x.new_empty(size, dtype=torch.uint8)
        _check(_on_device(device, h.expert_cache_adapt, self._at, x.data_ptr(), x.stride(0),
                          ids.data_ptr(), nbytes, T, base.data_ptr(), base.stride(0),
                          out.data_ptr(), out.stride(0), work.data_ptr()), "expert_cache_adapt")
        if given:
            _written(out)
        return out


# ---- pairs sorted by slot and back ---------------------------------------------------------

class Order:
    """Pairs of token and slot sorted by slot (`sort`). Pair t * k + j is token t's j-th.

    offsets  int32 [S + 1]: slot s has places offsets[s] to offsets[s + 1]
    rows     int32 [T * k]: the pair at every place, -1 from offsets[S] on
    places   int32 [T, k]: the place of every pair, -1 if its id is outside [0, S)"""

    __slots__ = ("offsets", "rows", "places", "T", "k", "S", "device")

    def __init__(self, offsets: torch.Tensor, rows: torch.Tensor, places: torch.Tensor, S: int):
        device = _on_gpu(offsets, rows, places)
        _need(places.dim() == 2 and 1 <= places.shape[1] <= MAX_TOP_K and
              places.numel() <= MAX_SORTED and 1 <= S <= MAX_EXPERTS and
              rows.shape == (places.numel(),) and offsets.shape == (S + 1,),
              f"offsets {list(offsets.shape)}, rows {list(rows.shape)} and places "
              f"{list(places.shape)} are no order of pairs by {S} slots")
        for t in (offsets, rows, places):
            _need(t.dtype == torch.int32 and t.is_contiguous(),
                  f"offsets, rows and places must be contiguous int32 on {device}")
        self._set(offsets, rows, places, S)

    def _set(self, offsets, rows, places, S):
        self.offsets, self.rows, self.places, self.S = offsets, rows, places, S
        self.T, self.k = places.shape
        self.device = places.device
        return self


def sort(slot_ids: torch.Tensor, slots: int) -> Order:
    """The pairs of token and slot, T x k int32 or int64 ids (or T of them: k is 1), slot by slot;
    those of a slot stay in the order of the tokens. Up to 1024 slots and 2^24 pairs, k up to 64."""
    shape = slot_ids.shape
    if len(shape) == 1:
        slot_ids, shape = slot_ids.unsqueeze(1), (shape[0], 1)
    if len(shape) != 2 or not 1 <= shape[1] <= MAX_TOP_K or shape[0] * shape[1] > MAX_SORTED:
        raise ValueError(f"slot_ids must be [T, k] or [T], k up to {MAX_TOP_K} and {MAX_SORTED} in "
                         f"all, not {list(shape)}")
    if not 1 <= slots <= MAX_EXPERTS:
        raise ValueError(f"{slots} slots (1 to {MAX_EXPERTS})")
    device = _on_gpu(slot_ids)
    ids, nbytes = _ids(slot_ids, device)
    T, k = shape
    n = T * k
    new = torch.empty(2 * n + slots + 1, dtype=torch.int32, device=device)
    rows, places, offsets = new.split((n, n, slots + 1))
    h = _lib.lib()
    size = _SORT_BYTES.get((n, slots))
    if size is None:
        need = ctypes.c_long()
        _check(h.expert_cache_sort_workspace(T, k, slots, ctypes.addressof(need)),
               "expert_cache_sort_workspace")
        if len(_SORT_BYTES) >= 4096:
            _SORT_BYTES.clear()
        size = _SORT_BYTES[n, slots] = need.value
    work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    _check(_on_device(device, h.expert_cache_sort, ids.data_ptr(), nbytes, T, k, slots,
                      offsets.data_ptr(), rows.data_ptr(), places.data_ptr(),
                      work.data_ptr() if size else None), "expert_cache_sort")
    return Order.__new__(Order)._set(offsets, rows, places.view(T, k), slots)


_SORT_BYTES: dict = {}  # workspace by pairs and slots


def _pitched(t: torch.Tensor) -> torch.Tensor:
    """`t` with its rows' values side by side and rows apart: itself, or a copy."""
    step = t.stride()
    return t if step[1] == 1 and (t.shape[0] < 2 or step[0] >= t.shape[1]) else t.contiguous()


def _movable(t, rows: int, order: Order, what: str) -> int:
    kind = _LOGITS.get(t.dtype)
    if kind is None or t.dim() != 2 or t.shape[0] != rows or t.device != order.device:
        raise ValueError(f"{what} must be float32, bfloat16 or float16 [{rows}, H] on "
                         f"{order.device}, not {t.dtype} {list(t.shape)} on {t.device}")
    if not 0 < t.shape[1] <= MAX_ROW:
        raise ValueError(f"rows of {t.shape[1]} (1 to {MAX_ROW})")
    if order.T * t.shape[1] * t.element_size() > MAX_MOVED:
        raise ValueError(f"{order.T} tokens of {t.shape[1]} {t.dtype} values ({MAX_MOVED} bytes)")
    return kind


def _recordable() -> None:
    if torch.cuda.is_current_stream_capturing():
        raise ValueError("a captured call cannot be recorded for a backward pass: capture it under "
                         "torch.no_grad(), with combine and combine_grad for the gradients")


def dispatch(x: torch.Tensor, order: Order) -> torch.Tensor:
    """The tokens' rows in the slots' order, [T * k, H]: row p is x[order.rows[p] // k], and rows
    from order.offsets[S] on are zeros. x [T, H] is float32, bfloat16 or float16; H up to 2^20, x up
    to 2^35 bytes.

    Differentiable in x, once: a token's gradient is the 32-bit sum of its rows', rounded to x's
    type. `combine(gradient, None, order)` is the same without autograd, for a call that is
    captured; one that autograd would record is refused then."""
    kind = _movable(x, order.T, order, "x")
    if forward_ad._current_level >= 0:
        _no_tangent(x)
    if x.requires_grad and torch.is_grad_enabled():
        _recordable()
        return _Dispatch.apply(x, order, kind)
    return _dispatch(x, order, kind)


def _dispatch(x, order, kind):
    x = _pitched(x)
    H, n = x.shape[1], order.T * order.k
    out = x.new_empty((n, H))
    _check(_on_device(order.device, _lib.lib().expert_cache_dispatch, x.data_ptr(), kind,
                      max(H, x.stride(0)), order.places.data_ptr(), order.rows.data_ptr(),
                      order.T, order.k, H, out.data_ptr(), H), "expert_cache_dispatch")
    return out


def combine(y: torch.Tensor, weights: torch.Tensor | None, order: Order) -> torch.Tensor:
    """Rows back to their tokens: [T, H], token t the sum over j of weights[t, j] times
    y[order.places[t, j]], in 32 bits and rounded to y's type. y [T * k, H] is float32, bfloat16 or
    float16, the result up to 2^35 bytes, weights float32 [T, k] or None (1). Pairs without a place or
    with a weight of 0 add nothing (and an infinity in their rows does not show).

    Differentiable in y and weights, once (`combine_grad` is the same without autograd, for a call
    that is captured; one that autograd would record is refused then)."""
    kind = _combine_args(y, weights, order)
    if forward_ad._current_level >= 0:
        _no_tangent(y, weights)
    if (y.requires_grad or (weights is not None and weights.requires_grad)) and \
            torch.is_grad_enabled():
        _recordable()
        return _Combine.apply(y, weights, order, kind)
    return _combine(y, weights, order, kind)


def _combine_args(y, weights, order) -> int:
    kind = _movable(y, order.T * order.k, order, "y")
    if weights is not None and (weights.dtype != torch.float32 or weights.device != order.device or
                                weights.shape != order.places.shape):
        raise ValueError(f"weights must be float32 {list(order.places.shape)} on {order.device}, "
                         f"not {weights.dtype} {list(weights.shape)} on {weights.device}")
    return kind


def _combine(y, weights, order, kind):
    y = _pitched(y)
    if weights is not None and not weights.is_contiguous():
        weights = weights.contiguous()
    H = y.shape[1]
    out = y.new_empty((order.T, H))
    _check(_on_device(order.device, _lib.lib().expert_cache_combine, y.data_ptr(), kind,
                      max(H, y.stride(0)), None if weights is None else weights.data_ptr(),
                      order.places.data_ptr(), order.T, order.k, H, out.data_ptr(), H),
           "expert_cache_combine")
    return out


def combine_grad(grad: torch.Tensor, y: torch.Tensor | None, weights: torch.Tensor | None,
                 order: Order, *, need_y: bool = True, need_weights: bool = True):
    """The gradients of `combine` from that of its result: (dy [T * k, H], dweights float32
    [T, k]), each None if it is not needed. dy[order.places[t, j]] is weights[t, j] * grad[t],
    rounded to its type, and zero from order.offsets[S] on; dweights[t, j] is the 32-bit dot product
    of grad[t] and y[order.places[t, j]], 0 without a place. y may be None without need_weights."""
    kind = _movable(grad, order.T, order, "grad")
    need_weights = need_weights and weights is not None
    if y is not None:
        _combine_args(y, weights, order)
        _need(y.shape[1] == grad.shape[1] and y.dtype == grad.dtype,
              f"y {y.dtype} {list(y.shape)} does not go with grad {grad.dtype} {list(grad.shape)}")
    else:
        _need(not need_weights, "the gradient of weights needs y")
        _need(weights is None or (weights.dtype == torch.float32 and
                                  weights.shape == order.places.shape and
                                  weights.device == order.device),
              f"weights must be float32 {list(order.places.shape)} on {order.device}")
    if forward_ad._current_level >= 0:
        _no_tangent(grad, y, weights)
    if torch.is_grad_enabled():
        _no_gradient(grad, y, weights)
    if not (need_y or need_weights):
        return None, None
    return _combine_grad(grad, y, weights, order, kind, need_y, need_weights)


def _combine_grad(grad, y, weights, order, kind, need_y, need_weights):
    H, n = grad.shape[1], order.T * order.k
    grad = _pitched(grad)
    y = _pitched(y) if need_weights else None
    dy = grad.new_empty((n, H)) if need_y else None
    dweights = grad.new_empty((order.T, order.k), dtype=torch.float32) if need_weights else None
    if weights is not None and not weights.is_contiguous():
        weights = weights.contiguous()
    _check(_on_device(order.device, _lib.lib().expert_cache_combine_grad, grad.data_ptr(), kind,
                      max(H, grad.stride(0)), None if y is None else y.data_ptr(),
                      H if y is None else max(H, y.stride(0)),
                      None if weights is None else weights.data_ptr(), order.places.data_ptr(),
                      order.rows.data_ptr(), order.T, order.k, H,
                      None if dy is None else dy.data_ptr(), H,
                      None if dweights is None else dweights.data_ptr()),
           "expert_cache_combine_grad")
    return dy, dweights


def _once(*tensors) -> None:
    if torch.is_grad_enabled():
        raise RuntimeError("dispatch and combine are differentiable once: their gradients have none "
                           "(create_graph)")
    if forward_ad._current_level >= 0:
        _no_tangent(*tensors)


# Autograd hands a result's gradient over in its shape and type, so `backward` checks neither again.

class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order, kind):
        ctx.of = order, kind
        return _dispatch(x, order, kind)

    @staticmethod
    def backward(ctx, grad):
        _once(grad)
        order, kind = ctx.of
        return _combine(grad, None, order, kind), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, order, kind):
        ctx.of = order, kind
        ctx.save_for_backward(y if ctx.needs_input_grad[1] else None, weights)
        return _combine(y, weights, order, kind)

    @staticmethod
    def backward(ctx, grad):
        y, weights = ctx.saved_tensors
        _once(grad, y, weights)
        order, kind = ctx.of
        need = ctx.needs_input_grad
        return *_combine_grad(grad, y, weights, order, kind, need[0], need[1]), None, None


# ---- products in 8-bit integers ------------------------------------------------------------

def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows as 8-bit integers and what 1 stands for: (q int8 [T, H], scales float32 [T]), with m a
    row's largest magnitude scales = m / 127 and q = 127 x / m to the nearest, ties to even. x is
    bfloat16 or float16 [T, H], T up to 2^23 and H 2^20; q's rows lie in ones of a multiple of 16. A
    row below 2^-119 throughout counts as zeros, and one with an infinity or NaN becomes zeros with a
    scale of NaN."""
    kind = _TOKENS.get(x.dtype)
    if kind is None or x.dim() != 2:
        raise ValueError(f"x must be bfloat16 or float16 [T, H], not {x.dtype} {list(x.shape)}")
    T, H = x.shape
    if T > MAX_TOKENS8 or not 0 < H <= MAX_ROW:
        raise ValueError(f"{T} rows (at most {MAX_TOKENS8}) of {H} (1 to {MAX_ROW})")
    device = _on_gpu(x)
    if forward_ad._current_level >= 0:
        _no_tangent(x)
    if torch.is_grad_enabled() and x.requires_grad:
        _no_gradient(x)
    x = _pitched(x)
    q = torch.empty((T, -(-H // 16) * 16), dtype=torch.int8, device=device)
    scales = torch.empty(T, dtype=torch.float32, device=device)
    _check(_on_device(device, _lib.lib().expert_cache_quantize, x.data_ptr(), kind,
                      max(H, x.stride(0)), T, H, q.data_ptr(), q.shape[1], scales.data_ptr()),
           "expert_cache_quantize")
    return q[:, :H] if q.shape[1] != H else q, scales


class Linear8:
    """A projection in 8-bit integers: y = x w^T + bias, tokens quantised with a scale each.

    w      int8 [O, H], H up to 131056, O 2^24        scale  float32 [O] or [O, 1], one a channel
    bias   float32, bfloat16 or float16 [O], or None

    Sums are exact; their product with both scales and the bias's sum are in 32 bits, and the result
    is rounded to its type. w is used as it lies if H and its rows are whole 16 bytes, and is copied
    otherwise, as is a bias that is not float32: a later change of those does not show."""

    def __init__(self, w: torch.Tensor, scale: torch.Tensor, bias: torch.Tensor | None = None):
        _need(w.dim() == 2 and w.dtype == torch.int8 and min(w.shape) > 0,
              f"w must be int8 [O, H], not {w.dtype} {list(w.shape)}")
        O, H = w.shape
        _need(H <= MAX_LENGTH8 and O <= MAX_SORTED,
              f"w {list(w.shape)} (at most [{MAX_SORTED}, {MAX_LENGTH8}])")
        self.device = _on_gpu(w, scale, bias)
        _scales(scale, (O,), "scale", self.device)
        if bias is not None:
            _need(bias.dtype in _LOGITS and bias.shape == (O,),
                  f"bias must be float32, bfloat16 or float16 [{O}], not {bias.dtype} "
                  f"{list(bias.shape)}")
        if forward_ad._current_level >= 0:
            _no_tangent(bias)  # a copy of it may be kept
        self._graded = _graded(w, scale, bias)
        step = w.stride()
        if H % 16 or w.data_ptr() % 16 or step[1] != 1 or \
                (O > 1 and (step[0] % 16 or step[0] < H or step[0] > 1 << 22)):
            laid = w.new_zeros((O, -(-H // 16) * 16))
            laid[:, :H] = w.detach()
            w = laid
        if bias is not None:
            bias = bias.detach().float().contiguous()
        self.w, self.scale, self.bias = w, scale, bias
        self.O, self.H = O, H
        self._struct = _lib.Linear(O, H, w.stride(0) if O > 1 else -(-H // 16) * 16, w.data_ptr(),
                                   scale.data_ptr(), None if bias is None else bias.data_ptr())
        self._at = ctypes.addressof(self._struct)
        self._bytes: dict = {}

    def __call__(self, x: torch.Tensor, x_scales: torch.Tensor | None = None, *,
                 dtype: torch.dtype | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        """[T, O] for tokens x [T, H] in bfloat16 or float16, or in int8 with x_scales float32 [T]
        as `quantize` makes them (projections that share their tokens quantise them once). The
        result's type is `dtype`: float32, bfloat16 or float16, if not given x's (bfloat16 for
        int8). `out`, if given, has contiguous rows and overlaps neither x nor x_scales."""
        kind = 3 if x.dtype == torch.int8 else _TOKENS.get(x.dtype)
        if kind is None or x.dim() != 2 or x.shape[1] != self.H or x.device != self.device:
            raise ValueError(f"x must be bfloat16, float16 or int8 [T, {self.H}] on {self.device}, "
                             f"not {x.dtype} {list(x.shape)} on {x.device}")
        T = x.shape[0]
        if T > MAX_TOKENS8 or T * self.O > MAX_RESULTS8:
            raise ValueError(f"{T} tokens (at most {MAX_TOKENS8}) of {self.O} results "
                             f"({MAX_RESULTS8} in all)")
        if dtype is None:
            dtype = torch.bfloat16 if kind == 3 else x.dtype
        to = _LOGITS.get(dtype)
        if to is None:
            raise ValueError(f"results of {dtype} (float32, bfloat16 or float16)")
        if (x_scales is None) != (kind != 3) or (x_scales is not None and (
                x_scales.dtype != torch.float32 or x_scales.shape != (T,) or
                x_scales.device != self.device)):
            raise ValueError(f"int8 tokens, and no others, have x_scales: float32 [{T}] on "
                             f"{self.device}")
        if forward_ad._current_level >= 0:
            _no_tangent(x, x_scales, out, self.scale, self.bias)
        if torch.is_grad_enabled() and (x.requires_grad or self._graded or out is not None or
                                        x_scales is not None):
            _no_gradient(x, x_scales, out, *self._graded)
        if kind == 3:
            x = self._whole(x)
            if not x_scales.is_contiguous():
                x_scales = x_scales.contiguous()
        else:
            x = _pitched(x)
        given = out is not None
        if not given:
            out = torch.empty((T, self.O), dtype=dtype, device=self.device)
        else:
            _out(out, dtype, (T, self.O), self.device)
        h, at = _lib.lib(), self._at
        size = self._bytes.get((kind == 3, T))
        if size is None:
            if len(self._bytes) >= 4096:
                self._bytes.clear()
            size = self._bytes[kind == 3, T] = _workspace(h.expert_cache_linear8_workspace, at, kind,
                                                          T)
        work = torch.empty(size, dtype=torch.uint8, device=self.device)
        _check(_on_device(self.device, h.expert_cache_linear8, at, x.data_ptr(), kind,
                          max(x.stride(0), self.H), None if kind != 3 else x_scales.data_ptr(), T,
                          out.data_ptr(), to, max(out.stride(0), self.O), work.data_ptr()),
               "expert_cache_linear8")
        if given:
            _written(out)
        return out

    def _whole(self, x: torch.Tensor) -> torch.Tensor:
        """8-bit rows that can be loaded 16 bytes at a time: `x`, or a copy."""
        step, length = x.stride(), -(-self.H // 16) * 16
        end = x.storage_offset() + (x.shape[0] - 1) * step[0] + length
        if x.shape[0] and (step[1] != 1 or x.data_ptr() % 16 or
                           end > x.untyped_storage().nbytes() or
                           (x.shape[0] > 1 and (step[0] % 16 or not length <= step[0] <= 1 << 22))):
            laid = x.new_zeros((x.shape[0], length))
            laid[:, :self.H] = x
            x = laid
        return x


class Experts8:
    """The experts of one layer, in slots or all of them, in 8-bit integers for any number of tokens.

    w13  int8 [S, 2*I, H]: gate rows, then up rows, w13_scale float32 [S, 2*I] or [S, 2*I, 1]
    w2   int8 [S, H, I], w2_scale float32 [S, H] or [S, H, 1]
    H and I are multiples of 16, S up to 1024.

    Tokens and hidden values are quantised row by row (`quantize`; hidden values from 32 bits), so
    results differ from `Experts`' by the rounding of those. Sums are exact, the rest is in 32 bits
    (the exponential of a gate value g to (2 |g| + 4) 2^-24 of itself, so a hidden value that near to
    half way between two whole numbers may go to either), the result is rounded to the tokens' type.
    The same call gives the same bits, and a token's are the same among any others. A token with an
    infinity or NaN gets NaN."""

    def __init__(self, w13: torch.Tensor, w2: torch.Tensor, w13_scale: torch.Tensor,
                 w2_scale: torch.Tensor):
        _need(w13.dim() == 3 and w2.dim() == 3 and w13.dtype == w2.dtype == torch.int8,
              "w13 and w2 must be int8 [S, 2*I, H] and [S, H, I]")
        S, two, H = w13.shape
        _need(two % 2 == 0 and tuple(w2.shape) == (S, H, two // 2) and min(S, two, H) > 0,
              f"w13 {list(w13.shape)} does not go with w2 {list(w2.shape)}")
        _need(H % 16 == 0 and (two // 2) % 16 == 0,
              f"H {H} and I {two // 2} must be multiples of 16")
        _need(max(H, two // 2) <= MAX_LENGTH8 and two * H <= MAX_BYTES8 and S <= MAX_EXPERTS,
              f"{S} slots (at most {MAX_EXPERTS}) of H {H} and I {two // 2} (at most {MAX_LENGTH8}, "
              f"w13 of {MAX_BYTES8} bytes)")
        for name, w in (("w13", w13), ("w2", w2)):
            _need(w.is_contiguous() and w.data_ptr() % 16 == 0,
                  f"{name} must be contiguous and 16-byte aligned")
        device = _on_gpu(w13, w2)
        _scales(w13_scale, (S, two), "w13_scale", device)
        _scales(w2_scale, (S, H), "w2_scale", device)
        self.w13, self.w2, self.w13_scale, self.w2_scale = w13, w2, w13_scale, w2_scale
        self.S, self.H, self.I, self.device = S, H, two // 2, device
        self._structs = {}
        for t, code in _TOKENS.items():
            e = _lib.Experts(S, H, two // 2, code, _BYTES[torch.int8], w13.data_ptr(),
                             w2.data_ptr(), w13_scale.data_ptr(), w2_scale.data_ptr())
            self._structs[t] = (e, ctypes.addressof(e))
        self._graded = _graded(w13_scale, w2_scale)
        self._bytes: dict = {}

    def __call__(self, x: torch.Tensor, topk_weights: torch.Tensor, slot_ids: torch.Tensor,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        """The layer's output [T, H] for tokens x [T, H] in bfloat16 or float16: the sum over their
        slots of the routing weight (float32 [T, top_k]) times the expert. slot_ids [T, top_k] are
        int32 or int64; T x top_k is at most 2^23, T x H 1.75 * 2^30. A pair whose id is outside
        [0, S) or whose weight is 0 adds nothing; a token without any other pair gets zeros. `out`,
        if given, has contiguous rows and overlaps no other argument."""
        struct = self._structs.get(x.dtype)
        if struct is None or x.dim() != 2 or x.shape[1] != self.H or x.device != self.device:
            raise ValueError(f"x must be bfloat16 or float16 [T, {self.H}] on {self.device}, not "
                             f"{x.dtype} {list(x.shape)} on {x.device}")
        T, shape = x.shape[0], slot_ids.shape
        if len(shape) != 2 or shape[0] != T or topk_weights.shape != shape or \
                topk_weights.dtype != torch.float32 or topk_weights.device != self.device:
            raise ValueError(f"slot_ids {list(shape)} and float32 topk_weights must be [{T}, top_k] "
                             f"on {self.device}, not {topk_weights.dtype} "
                             f"{list(topk_weights.shape)} on {topk_weights.device}")
        k = shape[1]
        if not 1 <= k <= MAX_TOP_K or T * k > MAX_TOKENS8 or T * self.H > MAX_BYTES8 or \
                T * k * max(self.H, self.I) > MAX_VALUES8:
            raise ValueError(f"{T} tokens of {self.H} x top_k {k} (top_k at most {MAX_TOP_K}, "
                             f"{MAX_TOKENS8} pairs, {MAX_BYTES8} values, {MAX_VALUES8} of the pairs')")
        if forward_ad._current_level >= 0:
            _no_tangent(x, topk_weights, out, self.w13, self.w2, self.w13_scale, self.w2_scale)
        if torch.is_grad_enabled() and (x.requires_grad or topk_weights.requires_grad or
                                        self._graded or out is not None):
            _no_gradient(x, topk_weights, out, *self._graded)
        ids, nbytes = _ids(slot_ids, self.device)
        if not topk_weights.is_contiguous():
            topk_weights = topk_weights.contiguous()
        x = _pitched(x)
        given = out is not None
        if not given:
            out = x.new_empty((T, self.H))
        else:
            _out(out, x.dtype, (T, self.H), self.device)
        h, at = _lib.lib(), struct[1]
        size = self._bytes.get((T, k))
        if size is None:
            if len(self._bytes) >= 4096:
                self._bytes.clear()
            size = self._bytes[T, k] = _workspace(h.expert_cache_moe8_workspace, at, T, k)
        work = x.new_empty(size, dtype=torch.uint8)
        _check(_on_device(self.device, h.expert_cache_moe8, at, x.data_ptr(),
                          max(x.stride(0), self.H), topk_weights.data_ptr(), ids.data_ptr(), nbytes,
                          T, k, out.data_ptr(), max(out.stride(0), self.H), work.data_ptr()),
               "expert_cache_moe8")
        if given:
            _written(out)
        return out

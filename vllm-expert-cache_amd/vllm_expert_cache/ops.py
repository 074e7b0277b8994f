"""Operators around the slot cache: the routing that makes its ids, and the products over what
its slots hold.

    weights, ids = route(logits, top_k)               # expert ids from the gate's logits
    slots = cache.refresh(ids)                        # experts into slots (cache.py)
    y = Experts(w13_slots, w2_slots)(x, weights, slots)

    slots = adapter_cache.refresh(adapter_ids)        # the same for adapters of requests
    y = Adapters(a_slots, b_slots)(x, projected, slots)

`Experts` and `Adapters` check their weights once and are kept like the weights themselves; a
cache's slot tensors never move, so a handle over them stays good. Weights are used as they lie,
without another layout. Calls run on the current stream of the tensors' device, allocate only
their result and a workspace through torch, and read nothing back, so they can be captured.

There is no backward pass: with gradients enabled, a tensor that requires one (a handle's weights:
when the handle is made) is refused.

ValueError names an argument that an operator does not take; nothing has run then.
"""
from __future__ import annotations

import ctypes

import torch

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


def _check(rc: int, name: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{name} failed rc={rc}")


# The current stream's handle without building a torch.cuda.Stream around it (a microsecond of
# each call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _on_device(device: torch.device, call, *args):
    """call(*args, stream) on the current stream of `device`, with that device current."""
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
        if torch.is_grad_enabled() and (x.requires_grad or topk_weights.requires_grad or
                                        self._graded or out is not None):
            _no_gradient(x, topk_weights, out, *self._graded)
        ids, nbytes = _ids(slot_ids, self.device)
        if not topk_weights.is_contiguous():
            topk_weights = topk_weights.contiguous()
        x = _rows(x)
        if out is None:
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
        return out


def _workspace(entry, struct, *sizes) -> int:
    size = ctypes.c_long()
    _check(entry(struct, *sizes, ctypes.addressof(size)), entry.__name__)
    return max(16, size.value)


def _out(out, dtype, shape, device) -> None:
    _need(out.dtype == dtype and tuple(out.shape) == shape and out.device == device and
          out.stride(1) == 1 and (shape[0] < 2 or out.stride(0) >= shape[1]),
          f"out must be {dtype} {list(shape)} on {device} with contiguous rows")


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
        if torch.is_grad_enabled() and (x.requires_grad or base.requires_grad or self._graded or
                                        out is not None):
            _no_gradient(x, base, out, *self._graded)
        ids, nbytes = _ids(slot_ids, device)
        x = _rows(x)
        if out is None:
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
        return out

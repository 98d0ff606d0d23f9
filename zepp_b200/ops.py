"""Operators around the expert-parallel layer, with gradients: what makes its ids and weights, and what trains its experts.

    ids, weights = route_topk(logits, k)                  # the gate
    rows, plan = sort_tokens(x, ids, num_experts)         # a row for every copy, by expert
    rows = expert_ffn(rows, plan.offsets, w1, w2)         # the experts' products and activation
    y = unsort_tokens(rows, plan, weights)                # back, with the weights applied
    norm = clip_grad_norm_(gradients, max_norm)           # the norm of all gradients, and clipping

Each call is one to five kernels of libzepp_b200.so on the current stream of its tensors' device; nothing is read back
on the host, and calls can be captured into CUDA graphs after one call on that device outside of a capture.  Arguments
that do not fit are refused with an AssertionError, as everywhere in this package.  Inputs that are not contiguous (or,
for expert_ffn, not on a 16-byte boundary) are copied.  Gradients are first derivatives only, and there are no forward-mode
derivatives: inputs that have a tangent are refused.

Where a backward pass is captured into a graph, make the forward pass that it belongs to inside the same capture, of
leaves that no graph outside of it still holds (torch runs a leaf's accumulation on the stream of the leaf's first use).
"""
import ctypes
import operator
import threading
from typing import NamedTuple

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ._ext import check, lib

__all__ = ["route_topk", "sort_tokens", "unsort_tokens", "SortPlan", "expert_ffn", "grad_norm", "clip_grad_norm_", "check_waits",
           "wait_failures", "set_wait_limit"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_SCORES = {"softmax": 0, "sigmoid": 1}
_ACTS = {"gelu": 0, "swiglu": 1}
MAX_GATE_EXPERTS, MAX_GATE_TOPK = 1024, 32
MAX_SORT_EXPERTS, MAX_SORT_TOPK = 2048, 64
MAX_FFN_EXPERTS = 1024
MAX_HIDDEN, MAX_ROWS = 1 << 20, (1 << 31) - 1      # of a row; of the sorted rows

_P, _I, _L, _F, _D = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float, ctypes.c_double
_ARGS = {
    "zepp_op_gate": (_P, _I, _L, _I, _I, _I, _I, _P, _F, _P, _P, _P),
    "zepp_op_gate_grad": (_P, _I, _L, _I, _I, _I, _I, _F, _P, _P, _P, _P, _P),
    "zepp_op_sort_ws_ints": (_L, _I, _I),
    "zepp_op_sort": (_P, _I, _L, _I, _L, _P, _P, _I, _I, _P, _P, _P, _P, _P),
    "zepp_op_unsort": (_P, _I, _L, _I, _L, _P, _P, _P, _P),
    "zepp_op_unsort_grad": (_P, _P, _I, _L, _I, _L, _I, _P, _P, _P, _P, _P, _P),
    "zepp_op_expert_ffn": (_P, _L, _P, _I, _I, _I, _I, _P, _P, _P, _P, _P, _P),
    "zepp_op_expert_ffn_grad": (_P, _P, _L, _P, _I, _I, _I, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P),
    "zepp_op_grad_norm_ws_bytes": (_I,),
    "zepp_op_grad_norm": (_P, _P, _P, _I, _D, _P, _P, _P),
    "zepp_op_set_wait_limit_ns": (_L,),
    "zepp_op_status": (_P, _P),
}
# a small call is bound by the host: these two cost a tenth of torch.cuda.current_device() and current_stream()
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_requires_grad = operator.attrgetter("requires_grad")
_SIZES = ("zepp_op_sort_ws_ints", "zepp_op_grad_norm_ws_bytes")
_fns = {}


def _fn(name):
    f = _fns.get(name)
    if f is None:
        f = getattr(lib(), name)
        f.argtypes = _ARGS[name]
        f.restype = ctypes.c_size_t if name in _SIZES else ctypes.c_int
        _fns[name] = f
    return f


def _refuse(what):
    raise AssertionError(what)


def _call(name, device, *args):
    """One entry point on the current stream of `device`."""
    index = device.index
    if index == _current_device():
        rc = _fn(name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = _fn(name)(*args, _raw_stream(index))
    if rc:
        check(rc)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _on(device, *tensors):
    for t in tensors:
        if t is not None and t.device != device:
            _refuse(f"a tensor is on {t.device}, not on {device} as the first one")


def _no_tangents(*tensors):
    """The kernels compute values only: of a dual tensor of forward-mode derivatives they would drop the tangent."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                _refuse("forward-mode derivatives: a tensor has a tangent, and the operators have gradients only")


def _first_derivative(backward):
    """once_differentiable, whose own cost (4 us) is paid only where a graph of the gradients is wanted"""
    slow = once_differentiable(backward)
    return staticmethod(lambda ctx, *grads: slow(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads))


# ------------------------------------------------------------------------------------------------ gate
def _gate(logits, k, score, renormalize, bias, scale):
    T, G = logits.shape
    weights = torch.empty((T, k), dtype=torch.float32, device=logits.device)
    ids = torch.empty_like(weights, dtype=torch.int32)
    _call("zepp_op_gate", logits.device, logits.data_ptr(), _TYPES[logits.dtype], T, G, k, score, renormalize, _ptr(bias),
          scale, ids.data_ptr(), weights.data_ptr())
    return ids, weights


class _Gate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, score, renormalize, bias, scale):
        ids, weights = _gate(logits, k, score, renormalize, bias, scale)
        ctx.save_for_backward(logits, ids, weights)
        ctx.how = (k, score, renormalize, scale)
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return ids, weights

    @_first_derivative
    def backward(ctx, _, dweights):
        if dweights is None:
            return (None,) * 6
        logits, ids, weights = ctx.saved_tensors
        k, score, renormalize, scale = ctx.how
        dlogits = torch.empty_like(logits)
        dweights = dweights.contiguous()
        _call("zepp_op_gate_grad", logits.device, logits.data_ptr(), _TYPES[logits.dtype], logits.shape[0], logits.shape[1], k,
              score, renormalize, scale, ids.data_ptr(), weights.data_ptr(), dweights.data_ptr(), dlogits.data_ptr())
        return dlogits, None, None, None, None, None


def route_topk(logits, k, score="softmax", renormalize=True, bias=None, scale=1.0):
    """The gate: ids [T, k] int32 of the k experts with the largest logits (largest first, equal ones by index) and their
    weights [T, k] float32, differentiable in the logits [T, E] (float32, bfloat16 or float16).

    score="softmax": a weight is the expert's probability over all experts; "sigmoid": the sigmoid of its logit.
    renormalize divides a token's weights by their sum; scale multiplies them.  bias [E] float32 (sigmoid only) is added
    to the scores for the choice alone and gets no gradient.  Experts whose logit is -inf or NaN are not chosen: a token
    that has fewer than k others gets id -1 and weight 0 in its last places (a token masked out altogether is a pad row of
    the layer).  A NaN in a row makes its weights NaN.  E <= 1024, k <= min(32, E)."""
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in _TYPES:
        _refuse(f"logits: a CUDA tensor [tokens, experts] of float32, bfloat16 or float16, got {tuple(logits.shape)} {logits.dtype} {logits.device}")
    G = logits.shape[1]
    if not 1 <= G <= MAX_GATE_EXPERTS or not 1 <= k <= min(MAX_GATE_TOPK, G):
        _refuse(f"1..{MAX_GATE_EXPERTS} experts and top-k of 1..min({MAX_GATE_TOPK}, experts), got {G} and {k}")
    if score not in _SCORES:
        _refuse(f"score: one of {tuple(_SCORES)}, got {score!r}")
    if bias is not None:
        if score != "sigmoid" or bias.shape != (G,) or bias.dtype != torch.float32:
            _refuse("bias: float32 [experts], with sigmoid scores")
        _on(logits.device, bias)
        bias = bias.detach().contiguous()
    _no_tangents(logits)
    logits = logits.contiguous()
    args = (logits, int(k), _SCORES[score], int(bool(renormalize)), bias, float(scale))
    return _Gate.apply(*args) if logits.requires_grad and torch.is_grad_enabled() else _gate(*args)


# ----------------------------------------------------------------------------------- sort by expert and back
class SortPlan(NamedTuple):
    """Where the copies of sort_tokens' tokens are: rows offsets[e] .. offsets[e + 1] belong to expert e (int32
    [experts + 1], the last one is the number of rows that hold a copy), position [T, K] int32 is a copy's row or -1."""
    offsets: torch.Tensor
    position: torch.Tensor


def _sort(x, ids, num_experts, group_of):
    T, K = ids.shape
    H = x.shape[1]
    rows = x.new_empty((T * K, H))
    offsets = ids.new_empty(num_experts + 1)
    position = torch.empty_like(ids)
    ints = _fn("zepp_op_sort_ws_ints")(T, K, num_experts)
    ws = ids.new_empty(ints) if ints else None
    _call("zepp_op_sort", x.device, x.data_ptr(), _TYPES[x.dtype], T, K, H, ids.data_ptr(), _ptr(group_of),
          0 if group_of is None else group_of.shape[0], num_experts, _ptr(ws), rows.data_ptr(), offsets.data_ptr(),
          position.data_ptr())
    return rows, offsets, position


def _unsort(rows, position, weights):
    T, K = position.shape
    H = rows.shape[1]
    y = rows.new_empty((T, H))
    _call("zepp_op_unsort", rows.device, rows.data_ptr(), _TYPES[rows.dtype], T, K, H, position.data_ptr(), _ptr(weights), y.data_ptr())
    return y


class _Sort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, num_experts, group_of):
        rows, offsets, position = _sort(x, ids, num_experts, group_of)
        ctx.save_for_backward(position)
        ctx.mark_non_differentiable(offsets, position)
        ctx.set_materialize_grads(False)
        return rows, offsets, position

    @_first_derivative
    def backward(ctx, drows, _offsets, _position):
        if drows is None:
            return None, None, None, None
        position, = ctx.saved_tensors
        return _unsort(drows.contiguous(), position, None), None, None, None


class _Unsort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, offsets, position, weights):
        ctx.save_for_backward(rows if weights is not None and ctx.needs_input_grad[3] else None, offsets, position, weights)
        ctx.like = (rows.shape, rows.dtype)
        return _unsort(rows, position, weights)

    @_first_derivative
    def backward(ctx, dy):
        rows, offsets, position, weights = ctx.saved_tensors
        dy = dy.contiguous()
        T, K = position.shape
        shape, dtype = ctx.like
        drows = dy.new_empty(shape) if ctx.needs_input_grad[0] else None
        dweights = torch.empty_like(weights) if ctx.needs_input_grad[3] else None
        _call("zepp_op_unsort_grad", dy.device, dy.data_ptr(), _ptr(rows), _TYPES[dtype], T, K, shape[1], offsets.shape[0] - 1,
              offsets.data_ptr(), position.data_ptr(), _ptr(weights), _ptr(drows), _ptr(dweights))
        return drows, None, None, dweights


def sort_tokens(x, ids, num_experts, group_of=None):
    """Rows of x [T, H] (float32, bfloat16 or float16), one for every copy, sorted by expert: (rows [T*K, H], SortPlan).
    Copies of an expert keep the order of (token, k).  ids [T, K] int32; a copy whose id is not one of the experts
    (the layer's pads have -1) gets no row, and rows that no copy fills are zero, at the end.  group_of: an int32 table
    that names the group of each id (such as a layer's slot of each expert); `num_experts` then counts groups.
    Differentiable in x.  K <= 64, H <= 2^20, at most 2048 experts, T*K < 2^31."""
    xs, s = x.shape, ids.shape
    if len(xs) != 2 or not x.is_cuda or x.dtype not in _TYPES or xs[1] < 1:
        _refuse(f"x: a CUDA tensor [tokens, hidden] of float32, bfloat16 or float16, got {tuple(x.shape)} {x.dtype} {x.device}")
    if len(s) != 2 or ids.dtype != torch.int32 or s[0] != xs[0] or not 1 <= s[1] <= MAX_SORT_TOPK:
        _refuse(f"ids: int32 [{xs[0]}, 1..{MAX_SORT_TOPK}], got {tuple(s)} {ids.dtype}")
    if xs[1] > MAX_HIDDEN or s[0] * s[1] > MAX_ROWS:
        _refuse(f"rows of at most {MAX_HIDDEN} elements, fewer than 2^31 copies, got {tuple(xs)} and {tuple(s)}")
    if not 1 <= num_experts <= MAX_SORT_EXPERTS:
        _refuse(f"1..{MAX_SORT_EXPERTS} experts, got {num_experts}")
    if group_of is not None:
        if group_of.dim() != 1 or group_of.dtype != torch.int32:
            _refuse("group_of: a table of int32")
        # an empty table has no address, which would stand for no table at all
        group_of = group_of.contiguous() if group_of.shape[0] else group_of.new_full((1,), -1)
    _on(x.device, ids, group_of)
    _no_tangents(x)
    args = (x.contiguous(), ids.contiguous(), int(num_experts), group_of)
    rows, offsets, position = _Sort.apply(*args) if x.requires_grad and torch.is_grad_enabled() else _sort(*args)
    return rows, SortPlan(offsets, position)


def unsort_tokens(rows, plan, weights=None):
    """The inverse of sort_tokens: y [T, H], y[t] = sum over k of weights[t, k] * rows[plan.position[t, k]] over the copies
    that have a row, added up in float32 in the order of k.  weights [T, K] float32; without them every copy counts once.
    Differentiable in rows and weights."""
    T, K = plan.position.shape
    s = rows.shape
    if len(s) != 2 or not rows.is_cuda or rows.dtype not in _TYPES or s[0] != T * K or s[1] < 1:
        _refuse(f"rows: [{T * K}, hidden] of float32, bfloat16 or float16, got {tuple(s)} {rows.dtype} {rows.device}")
    if s[1] > MAX_HIDDEN or s[0] > MAX_ROWS:
        _refuse(f"rows of at most {MAX_HIDDEN} elements, fewer than 2^31 of them, got {tuple(s)}")
    if plan.position.dtype != torch.int32 or plan.offsets.dtype != torch.int32 or not 1 <= K <= MAX_SORT_TOPK:
        _refuse("plan: as sort_tokens returns it")
    if weights is not None:
        if weights.shape != (T, K) or weights.dtype != torch.float32:
            _refuse(f"weights: float32 [{T}, {K}], got {tuple(weights.shape)} {weights.dtype}")
        weights = weights.contiguous()
    _on(rows.device, plan.position, plan.offsets, weights)
    _no_tangents(rows, weights)
    rows = rows.contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad)):
        return _Unsort.apply(rows, plan.offsets.contiguous(), plan.position.contiguous(), weights)
    return _unsort(rows, plan.position.contiguous(), weights)


# -------------------------------------------------------------------------------------------- experts' products
def _dense16(t):
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _ffn(rows, offsets, w1, w2, act, keep):
    n, H = rows.shape
    G, f1 = w1.shape[:2]
    I = w2.shape[2]
    y = torch.empty_like(rows)
    a = rows.new_empty((n, I))
    h = torch.empty((n, f1), dtype=torch.float32, device=rows.device) if keep else None
    _call("zepp_op_expert_ffn", rows.device, rows.data_ptr(), n, offsets.data_ptr(), G, H, I, act, w1.data_ptr(), w2.data_ptr(),
          a.data_ptr(), _ptr(h), y.data_ptr())
    return y, a, h


class _ExpertFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, offsets, w1, w2, act):
        y, a, h = _ffn(rows, offsets, w1, w2, act, True)
        ctx.save_for_backward(rows, offsets, w1, w2, a, h)
        ctx.act = act
        return y

    @_first_derivative
    def backward(ctx, dy):
        rows, offsets, w1, w2, a, h = ctx.saved_tensors
        n, H = rows.shape
        G, f1 = w1.shape[:2]
        need = ctx.needs_input_grad
        dy = _dense16(dy)
        drows = torch.empty_like(rows) if need[0] else None
        dw1 = torch.empty_like(w1) if need[2] else None
        dw2 = torch.empty_like(w2) if need[3] else None
        dh = rows.new_empty((n, f1)) if need[0] or need[2] else None
        _call("zepp_op_expert_ffn_grad", rows.device, dy.data_ptr(), rows.data_ptr(), n, offsets.data_ptr(), G, H, w2.shape[2],
              ctx.act, w1.data_ptr(), w2.data_ptr(), a.data_ptr(), h.data_ptr(), _ptr(dh), _ptr(drows), _ptr(dw1), _ptr(dw2))
        return drows, None, dw1, dw2, None


def expert_ffn(rows, offsets, w1, w2, act="swiglu"):
    """Each expert's two products and the activation between them on its own rows: y [n, H] of rows [n, H], where rows
    offsets[e] .. offsets[e + 1] go through w1[e] [ffn1, H] and w2[e] [H, ffn] (ffn1 = 2 ffn for "swiglu": gate rows, then
    up rows, as the layer holds them; ffn for "gelu").  All bfloat16, accumulated in float32; offsets int32 [experts + 1]
    on the device, not decreasing, starting at 0; rows behind the last expert's give zero.  hidden and ffn are
    multiples of 8, up to 2^20 and 2^19; at most 1024 experts, fewer than 2^31 rows.  Differentiable in rows, w1 and w2; an
    expert without rows has a zero gradient."""
    if act not in _ACTS:
        _refuse(f"act: one of {tuple(_ACTS)}, got {act!r}")
    if not rows.is_cuda or rows.dim() != 2 or w1.dim() != 3 or w2.dim() != 3:
        _refuse(f"rows [n, hidden], w1 [experts, ffn1, hidden], w2 [experts, hidden, ffn] on a GPU, got {tuple(rows.shape)}, "
                f"{tuple(w1.shape)}, {tuple(w2.shape)} on {rows.device}")
    G, H, I = w2.shape
    if rows.shape[1] != H or w1.shape != (G, I * (2 if act == "swiglu" else 1), H) or offsets.shape != (G + 1,):
        _refuse(f"shapes do not fit: rows {tuple(rows.shape)}, w1 {tuple(w1.shape)}, w2 {tuple(w2.shape)}, offsets {tuple(offsets.shape)}, {act}")
    if rows.dtype != torch.bfloat16 or w1.dtype != torch.bfloat16 or w2.dtype != torch.bfloat16 or offsets.dtype != torch.int32:
        _refuse("rows and weights are bfloat16, offsets int32")
    if H % 8 or I % 8 or H < 8 or I < 8 or not 1 <= G <= MAX_FFN_EXPERTS:
        _refuse(f"hidden and ffn are multiples of 8, 1..{MAX_FFN_EXPERTS} experts, got {H}, {I}, {G}")
    if H > MAX_HIDDEN or I > MAX_HIDDEN // 2 or rows.shape[0] > MAX_ROWS:
        _refuse(f"hidden up to {MAX_HIDDEN}, ffn up to {MAX_HIDDEN // 2}, fewer than 2^31 rows, got {H}, {I}, {rows.shape[0]}")
    _on(rows.device, offsets, w1, w2)
    _no_tangents(rows, w1, w2)
    args = (_dense16(rows), offsets.contiguous(), _dense16(w1), _dense16(w2), _ACTS[act])
    if torch.is_grad_enabled() and (rows.requires_grad or w1.requires_grad or w2.requires_grad):
        return _ExpertFFN.apply(*args)
    return _ffn(*args, False)[0]


# ---------------------------------------------------------------------------------- norm of all gradients, clipping
def _is_dense(t):
    """Every element of the tensor's span belongs to it once, whatever the order of its dimensions."""
    need = 1
    for stride, size in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n != 1):
        if stride != need:
            return False
        need *= size
    return True


def _norm(tensors, max_norm):
    tensors = list(tensors)
    if not tensors:
        _refuse("no tensors")
    device = tensors[0].device
    dtypes = [t.dtype for t in tensors]
    kinds = set(dtypes)
    if device.type != "cuda" or not _TYPES.keys() >= kinds or set(map(torch.Tensor.get_device, tensors)) != {device.index}:
        _refuse("CUDA tensors of one device, of float32, bfloat16 or float16")
    if not all(map(torch.Tensor.is_contiguous, tensors)) and not all(t.is_contiguous() or _is_dense(t) for t in tensors):
        _refuse("tensors whose elements lie without gaps and only once in memory")
    if forward_ad._current_level >= 0:
        _no_tangents(*tensors)
    n = len(tensors)
    out = torch.empty((), dtype=torch.float32, device=device)
    ws = torch.empty(_fn("zepp_op_grad_norm_ws_bytes")(n), dtype=torch.uint8, device=device)
    # Short lists in plain Python, long ones in numpy, whose calls have a fixed cost. Host time of a clipping call, plain
    # against numpy: 19 and 29 us for 1 tensor, 25 and 33 for 8, 30 and 36 for 16; of a norm alone 17 and 21, 21 and 23, 25 and 25.
    if n <= 16:
        ptrs, sizes, types = [t.data_ptr() for t in tensors], [t.numel() for t in tensors], [_TYPES[d] for d in dtypes]
        if max_norm >= 0:
            spans = sorted((p, p + c * (2 if ty else 4)) for p, c, ty in zip(ptrs, sizes, types) if c)
            overlap = any(b[0] < a[1] for a, b in zip(spans, spans[1:]))
        tables = (_P * n)(*ptrs), (_L * n)(*sizes), (ctypes.c_uint8 * n)(*types)
        at = [ctypes.addressof(t) for t in tables]
    else:
        ptrs = np.fromiter(map(torch.Tensor.data_ptr, tensors), np.uint64, n)
        sizes = np.fromiter(map(torch.Tensor.numel, tensors), np.uint64, n)      # the same bytes as int64
        if len(kinds) == 1:
            types = np.full(n, _TYPES[dtypes[0]], np.uint8)
        else:
            types = np.fromiter(map(_TYPES.__getitem__, dtypes), np.uint8, n)
        if max_norm >= 0:
            first, last = ptrs, ptrs + sizes * (np.uint64(4) >> (types != 0))
            some = sizes != 0
            if not some.all():
                first, last = first[some], last[some]
            if (first[1:] < last[:-1]).any():              # not one behind the other as they are
                order = first.argsort()
                overlap = (first[order[1:]] < last[order[:-1]]).any()
            else:
                overlap = False
        at = [t.ctypes.data for t in (ptrs, sizes, types)]
    if max_norm >= 0 and overlap:
        _refuse("tensors that do not overlap (one is given twice?)")
    _call("zepp_op_grad_norm", device, *at, n, max_norm, out.data_ptr(), ws.data_ptr())
    return out


def grad_norm(tensors):
    """The 2-norm over all elements of the tensors (float32, bfloat16 and float16 may be mixed), a float32 scalar on their
    device; sums run in 64 bits across chunks and in a fixed order.  Not differentiable."""
    return _norm(tensors, -1.0)


def clip_grad_norm_(tensors, max_norm):
    """Scale the tensors in place by min(1, max_norm / (norm + 1e-6)), norm being grad_norm(tensors), which is returned.
    The tensors are the gradients themselves, not parameters: leaves that require a gradient are refused.
    With a norm of NaN every element becomes NaN; where an element is infinite, the finite ones become 0 and the infinite ones
    NaN; with an infinite max_norm only NaN changes anything.  The tensors must not overlap; other orders of their dimensions
    are fine, gaps are not."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        _refuse(f"max_norm: not negative, got {max_norm}")
    tensors = list(tensors)
    if any(map(_requires_grad, tensors)) and any(t.requires_grad and t.is_leaf for t in tensors):
        _refuse("gradients, not the parameters that they belong to: a tensor is a leaf that requires a gradient")
    out = _norm(tensors, max_norm)
    torch.autograd.graph.increment_version(tensors)      # graphs that saved a tensor learn that it changed
    return out


def set_wait_limit(seconds):
    """How long a bounded wait of the operators' kernels lasts before the kernel gives up, for calls from now on (2 s where
    nothing was set; captured graphs keep the limit that they were captured with)."""
    if not 0 <= seconds <= 3600:
        _refuse(f"a wait limit of 0..3600 seconds, got {seconds}")
    check(_fn("zepp_op_set_wait_limit_ns")(int(seconds * 1e9)))


_waits = {}                       # device ordinal: [failures read so far, the last one's words, those that check_waits has raised for]
_waits_lock = threading.Lock()


def _status(index):
    """The operators' status words of a device; a failure is cleared there as it is read."""
    out = (ctypes.c_uint64 * 8)()
    with torch.cuda.device(index):
        check(_fn("zepp_op_status")(_raw_stream(index), ctypes.addressof(out)))
    return list(out)


def _device_index(device):
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        _refuse(f"a CUDA device, got {device}")
    return _current_device() if device.index is None else device.index


def _wait_report(index):
    words = _waits[index][1]
    return f"zepp_b200 operator failed: a device-side wait ran out (wait id {words[1]}, item {words[2]}, step {words[3]})"


def wait_failures(device=None):
    """How many times, since the process began, a look at the device (default: the current one) has found that a bounded wait
    of an operator's kernel had run out; looks once more first, after synchronising the device.  Nobody's look takes a
    failure away from another: each compares the count with its own last one."""
    index = _device_index(device)
    with _waits_lock:
        words = _status(index)
        seen = _waits.setdefault(index, [0, None, 0])
        if words[0]:
            seen[0] += 1
            seen[1] = words
        return seen[0]


def check_waits(device=None):
    """Synchronise the device (default: the current one) and raise if a bounded wait of an operator's kernel on it, on any
    stream, has run out since the last check_waits: outputs of the calls in between may be incomplete."""
    index = _device_index(device)
    count = wait_failures(index)
    seen = _waits[index]
    if count > seen[2]:
        seen[2] = count
        raise RuntimeError(_wait_report(index))

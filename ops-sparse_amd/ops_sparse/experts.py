"""The experts' operators on torch tensors: routing, ragged products grouped by expert, their combination.

T tokens each choose k of E experts.  The choice is a CSR matrix of k entries per row; :class:`ExpertPlan` is its
pattern by columns, which the products read.  One layer is::

    weights, ids, plan = route(x @ gate.T, k)               # the router
    h = grouped_mm(x, w_in, plan, gather=True)              # row r: w_in[e] @ x[token of r], e the expert of row r
    y = combine(grouped_mm(act(h), w_out, plan), plan, weights)

``weights``, the products and the combination are differentiable.  Everything runs through libaclsparse_hip.so on
the current torch stream; nothing waits for the device.  There is no CPU path.  The reference has no counterpart.
"""
import ctypes
import functools
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import Operation, check
from .spmv import Handle, acl_dtype

_MAX_EXPERTS, _MAX_K = 1024, 64
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
_HALVES = (torch.float16, torch.bfloat16)


class ExpertPlan(NamedTuple):
    """The assignments of tokens to experts, sorted by expert (int32 tensors on the device).

    offsets [E + 1]: rows offsets[e] to offsets[e + 1] are expert e's; tokens [T * k]: the token of each row (-1
    past offsets[E]); places [T, k]: the row of each assignment, -1 for a dropped one.  ``tokens`` and ``places``
    may be None where rows are grouped by other means: such a plan serves products that do not gather.
    """
    offsets: torch.Tensor
    tokens: Optional[torch.Tensor] = None
    places: Optional[torch.Tensor] = None


# the C enumeration's value of each type (a dictionary look-up costs less than an enumeration's conversion)
_TYPE = {t: int(acl_dtype(t)) for t in (torch.float32, torch.float16, torch.bfloat16, torch.int8)}
_NN, _NT = int(Operation.NON_TRANSPOSE), int(Operation.TRANSPOSE)

# torch's own look-ups of the current stream and device without the objects that its public ones build around
# them (4 us of a call's 14); the public ones where a version has not got them
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device

_HANDLES = {}
_FUNCTIONS = {}


def _call(device, name, *args):
    """Calls a C function on the device's current stream, with that device current.

    Handles are kept per stream: one holds nothing but the stream.
    """
    index = device.index
    stream = _raw_stream(index) or _lib.HIP_NULL_STREAM
    handle = _HANDLES.get((index, stream))
    if handle is None:
        handle = _HANDLES[(index, stream)] = Handle(stream)
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = getattr(_lib.lib(), name)
    if _current_device() == index:
        status = fn(handle.h, *args)
    else:
        with torch.cuda.device(device):
            status = fn(handle.h, *args)
    if status:
        check(name, status)


def _tracked(*tensors):
    """Whether autograd has to see the call."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _on_device(first, **others):
    if not first.is_cuda:
        raise ValueError("the experts' operators need tensors on a ROCm device")
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{name} must be on {first.device}, got {t.device}")


def _rows(t):
    """t with its last dimension contiguous and rows that do not overlap (a copy only where it is not so)."""
    if t.stride(-1) == 1 or t.shape[-1] <= 1:
        if t.dim() < 2 or t.shape[-2] <= 1 or t.stride(-2) >= t.shape[-1]:
            return t
    return t.contiguous()


def _ld(t):
    return max(t.stride(-2), t.shape[-1], 1) if t.shape[-2] > 1 else max(t.shape[-1], 1)


def _index(t, name):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    return t.contiguous()


def _plan_args(plan, gather, device):
    offsets, tokens = _index(plan.offsets, "offsets"), plan.tokens
    if offsets.dim() != 1 or offsets.numel() < 2:
        raise ValueError("offsets must be one-dimensional, one more than the experts")
    if gather:
        if tokens is None:
            raise ValueError("gather needs the plan's tokens")
        tokens = _index(tokens, "tokens")
    for name, t in (("offsets", offsets), ("tokens", tokens if gather else None)):
        if t is not None and t.device != device:
            raise ValueError(f"{name} must be on {device}, got {t.device}")
    return offsets, tokens if gather else None


# ---------------------------------------------------------------------------------------------------- routing


def _route_shape(tokens, experts, k):
    if not 1 <= k <= experts:
        raise ValueError(f"k must lie in [1, {experts}], got {k}")
    if experts > _MAX_EXPERTS or k > _MAX_K:
        raise ValueError(f"at most {_MAX_EXPERTS} experts and k <= {_MAX_K}, got {experts} and {k}")
    if tokens * k > 2**31 - 1:
        raise ValueError("tokens * k must fit int32")


@functools.lru_cache(maxsize=256)
def _buffer_size(device, tokens, experts, k):
    size = ctypes.c_size_t(0)
    _call(device, "aclsparseRoute_bufferSize", tokens, experts, k, ctypes.byref(size))
    return size.value


def _plan_tensors(tokens, experts, k, device, ids):
    """Plan tensors (with the choice's where ``ids``) and the buffer of a routing call, in one allocation."""
    n = tokens * k
    sizes = [n, n, n if ids else 0, experts + 1, _buffer_size(device, tokens, experts, k) // 4]
    starts = [0]
    for size in sizes:
        starts.append(starts[-1] + (size + 15) // 16 * 16)  # each part at a multiple of 64 bytes
    data = torch.empty(starts[-1], dtype=torch.int32, device=device)
    row_tokens = data.as_strided((n,), (1,), starts[0])
    places = data.as_strided((tokens, k), (k, 1), starts[1])
    chosen = data.as_strided((tokens, k), (k, 1), starts[2]) if ids else None
    offsets = data.as_strided((experts + 1,), (1,), starts[3])
    return offsets, row_tokens, places, chosen, data.data_ptr() + 4 * starts[4]


def _route(logits, k, normalize):
    tokens, experts = logits.shape
    offsets, row_tokens, places, ids, buffer = _plan_tensors(tokens, experts, k, logits.device, True)
    weights = torch.empty(tokens, k, dtype=torch.float32, device=logits.device)
    _call(logits.device, "aclsparseRoute", tokens, experts, k, logits.data_ptr(), _ld(logits), _TYPE[logits.dtype],
          int(normalize), weights.data_ptr(), ids.data_ptr(), offsets.data_ptr(), row_tokens.data_ptr(),
          places.data_ptr(), buffer)
    return weights, ids, offsets, row_tokens, places


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, normalize):
        logits = _rows(logits)
        weights, ids, offsets, row_tokens, places = _route(logits, k, normalize)
        ctx.mark_non_differentiable(ids, offsets, row_tokens, places)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(None if normalize else logits, weights, ids)
        ctx.dtype, ctx.shape, ctx.normalize = logits.dtype, logits.shape, normalize
        return weights, ids, offsets, row_tokens, places

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad, *_unused):
        if grad is None:
            return None, None, None
        logits, weights, ids = ctx.saved_tensors
        tokens, experts = ctx.shape
        grad = grad.to(torch.float32).contiguous()
        out = torch.empty(tokens, experts, dtype=ctx.dtype, device=ids.device)
        _call(ids.device, "aclsparseRouteGrad", tokens, experts, ids.shape[1],
              logits.data_ptr() if logits is not None else None, _ld(logits) if logits is not None else 0,
              _TYPE[ctx.dtype], int(ctx.normalize), weights.data_ptr(), ids.data_ptr(), grad.data_ptr(),
              out.data_ptr(), experts)
        return out, None, None


def route(logits, k, normalize=True):
    """(weights, ids, plan) of router logits [T, E] (fp32, fp16 or bf16): the k largest of each row, ties to the
    lowest index, never -inf (such a choice has id -1, weight 0 and place -1; NaN counts as the largest).

    weights [T, k] fp32 (differentiable): exp(l_j - max) / sum, the sum over the chosen or, with ``normalize`` false,
    over the row; ids [T, k] int32, largest first; plan: the assignments sorted by expert.
    """
    if logits.dim() != 2:
        raise ValueError("logits must be two-dimensional")
    if logits.dtype not in _FLOATS:
        raise TypeError(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    _on_device(logits)
    _route_shape(logits.shape[0], logits.shape[1], k)
    if _tracked(logits):
        weights, ids, offsets, tokens, places = _Route.apply(logits, k, bool(normalize))
    else:
        weights, ids, offsets, tokens, places = _route(_rows(logits), k, bool(normalize))
    return weights, ids, ExpertPlan(offsets, tokens, places)


def expert_plan(ids, experts):
    """The plan of a given choice: ids [T, k] int32, those outside [0, experts) dropped."""
    if ids.dim() != 2:
        raise ValueError("ids must be two-dimensional")
    _on_device(ids)
    ids = _index(ids, "ids")
    tokens, k = ids.shape
    if k < 1 or experts < 1:
        raise ValueError("there must be one choice and one expert at least")
    if k > min(experts, _MAX_K) or experts > _MAX_EXPERTS or tokens * k > 2**31 - 1:
        raise ValueError(f"at most {_MAX_EXPERTS} experts and k <= {_MAX_K} and the experts, got {experts} and {k}")
    offsets, row_tokens, places, _, buffer = _plan_tensors(tokens, experts, k, ids.device, False)
    _call(ids.device, "aclsparseExpertPlan", tokens, experts, k, ids.data_ptr(), offsets.data_ptr(),
          row_tokens.data_ptr(), places.data_ptr(), buffer)
    return ExpertPlan(offsets, row_tokens, places)


# ---------------------------------------------------------------------------------------------------- products


def _grouped(op, a, b, offsets, index, rows, n, k, out_dtype):
    out = torch.empty(rows, n, dtype=out_dtype, device=a.device)
    _call(a.device, "aclsparseGroupedMM", op, b.shape[0], rows, n, k, offsets.data_ptr(),
          index.data_ptr() if index is not None else None, a.shape[0], a.data_ptr(), _ld(a), b.data_ptr(), _ld(b),
          b.stride(0) if b.shape[0] > 1 else 0, _TYPE[a.dtype], out.data_ptr(), max(n, 1),
          _TYPE[out_dtype])
    return out


def _combine(y, places, weights, dtype):
    tokens, k = places.shape
    out = torch.empty(tokens, y.shape[1], dtype=dtype, device=y.device)
    _call(y.device, "aclsparseCombine", tokens, k, y.shape[1], y.shape[0], places.data_ptr(),
          weights.data_ptr() if weights is not None else None, y.data_ptr(), _ld(y), _TYPE[y.dtype],
          out.data_ptr(), max(y.shape[1], 1), _TYPE[dtype])
    return out


class _GroupedMM(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, w, offsets, tokens, places):
        a, w = _rows(a), _rows(w)
        rows = a.shape[0] if tokens is None else tokens.numel()
        ctx.save_for_backward(a, w, offsets, tokens, places)
        return _grouped(_NT, a, w, offsets, tokens, rows, w.shape[1], w.shape[2], a.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        a, w, offsets, tokens, places = ctx.saved_tensors
        grad = _rows(grad)
        rows, (groups, n, k) = grad.shape[0], w.shape
        da = dw = None
        if ctx.needs_input_grad[0]:
            if tokens is None:
                da = _grouped(_NN, grad, w, offsets, None, rows, k, n, a.dtype)
            else:
                # a token's rows are summed in fp32 and rounded once
                part = _grouped(_NN, grad, w, offsets, None, rows, k, n, torch.float32)
                da = _combine(part, places, None, a.dtype)
        if ctx.needs_input_grad[1]:
            dw = torch.empty(groups, n, k, dtype=w.dtype, device=w.device)
            _call(a.device, "aclsparseGroupedMMGrad", groups, rows, n, k, offsets.data_ptr(),
                  tokens.data_ptr() if tokens is not None else None, a.shape[0], grad.data_ptr(), _ld(grad),
                  a.data_ptr(), _ld(a), _TYPE[a.dtype], dw.data_ptr(), max(k, 1), n * k,
                  _TYPE[dw.dtype])
        return da, dw, None, None, None


def grouped_mm(a, w, plan, gather=False):
    """y [R, N]: y[r] = w[e] @ a[r] for the rows r of each expert e, rows past the last expert's zero (differentiable).

    w [E, N, K], fp16 or bf16 (any strides whose last is 1 avoid a copy); a of its type: [R, K] in the plan's row
    order or, with ``gather``, [T, K] in token order: row r then reads a[plan.tokens[r]].  Sums are in fp32.
    """
    if a.dim() != 2 or w.dim() != 3 or a.shape[1] != w.shape[2]:
        raise ValueError(f"a must be [rows, K] and w [experts, N, K], got {tuple(a.shape)} and {tuple(w.shape)}")
    if a.dtype not in _HALVES or w.dtype != a.dtype:
        raise TypeError(f"a and w must both be float16 or bfloat16, got {a.dtype} and {w.dtype}")
    _on_device(a, w=w)
    offsets, tokens = _plan_args(plan, gather, a.device)
    if offsets.numel() != w.shape[0] + 1:
        raise ValueError(f"the plan has {offsets.numel() - 1} experts, w {w.shape[0]}")
    if not _tracked(a, w):
        a, w = _rows(a), _rows(w)
        return _grouped(_NT, a, w, offsets, tokens, a.shape[0] if tokens is None else tokens.shape[0], w.shape[1],
                        w.shape[2], a.dtype)
    places = None
    if gather and a.requires_grad:
        if plan.places is None or plan.places.numel() != tokens.numel() or plan.places.shape[0] != a.shape[0]:
            raise ValueError("a gradient through gather needs the plan's places, [tokens, k]")
        places = _index(plan.places, "places")
    return _GroupedMM.apply(a, w, offsets, tokens, places)


def grouped_mm_scaled(a, a_scale, w, w_scale, plan=None, gather=False, out_dtype=torch.bfloat16):
    """:func:`grouped_mm` of 8-bit integers: y[r, n] = a_scale[i] * w_scale[e, n] * (the exact integer product), i the
    row of a that row r reads.  a int8, a_scale [rows of a] fp32, w [E, N, K] int8, w_scale [E, N] fp32; with no plan
    one dense product, w [N, K] and w_scale [N].  K <= 131071, so that the sum stays within 32 bits.  No gradient.
    """
    dense = plan is None
    if dense:
        if gather:
            raise ValueError("gather needs a plan")
        if w.dim() != 2 or w_scale.dim() != 1:
            raise ValueError("without a plan w is [N, K] and w_scale [N]")
        w, w_scale = w.unsqueeze(0), w_scale.unsqueeze(0)
    if a.dim() != 2 or w.dim() != 3 or a.shape[1] != w.shape[2]:
        raise ValueError(f"a must be [rows, K] and w [experts, N, K], got {tuple(a.shape)} and {tuple(w.shape)}")
    if a.dtype != torch.int8 or w.dtype != torch.int8:
        raise TypeError(f"a and w must be int8, got {a.dtype} and {w.dtype}")
    if a_scale.dtype != torch.float32 or w_scale.dtype != torch.float32:
        raise TypeError("the scales must be float32")
    if tuple(a_scale.shape) != (a.shape[0],) or tuple(w_scale.shape) != tuple(w.shape[:2]):
        raise ValueError("a_scale must hold one scale per row of a, w_scale one per row of w")
    if out_dtype not in _FLOATS:
        raise TypeError(f"out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    if a.shape[1] > 131071:
        raise ValueError("K must not exceed 131071")
    _on_device(a, a_scale=a_scale, w=w, w_scale=w_scale)
    a, w, a_scale, w_scale = _rows(a), _rows(w), a_scale.contiguous(), w_scale.contiguous()
    offsets = tokens = None
    if not dense:
        offsets, tokens = _plan_args(plan, gather, a.device)
        if offsets.numel() != w.shape[0] + 1:
            raise ValueError(f"the plan has {offsets.numel() - 1} experts, w {w.shape[0]}")
    rows = a.shape[0] if tokens is None else tokens.numel()
    groups, n, k = w.shape
    out = torch.empty(rows, n, dtype=out_dtype, device=a.device)
    _call(a.device, "aclsparseGroupedMMScaled", groups, rows, n, k, offsets.data_ptr() if offsets is not None else None,
          tokens.data_ptr() if tokens is not None else None, a.shape[0], a.data_ptr(), _ld(a), a_scale.data_ptr(),
          w.data_ptr(), _ld(w), w.stride(0) if groups > 1 else 0, w_scale.data_ptr(), out.data_ptr(), max(n, 1),
          _TYPE[out_dtype])
    return out


# ---------------------------------------------------------------------------------------------------- combination


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, offsets, places):
        y = _rows(y)
        ctx.save_for_backward(y, weights, offsets, places)
        return _combine(y, places, weights, y.dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        y, weights, offsets, places = ctx.saved_tensors
        grad = _rows(grad)
        tokens, k = places.shape
        rows, width = y.shape
        dy = torch.empty(rows, width, dtype=y.dtype, device=y.device) if ctx.needs_input_grad[0] else None
        dw = torch.empty(tokens, k, dtype=torch.float32, device=y.device) if ctx.needs_input_grad[1] else None
        _call(y.device, "aclsparseCombineGrad", tokens, k, width, rows, offsets.numel() - 1, offsets.data_ptr(),
              places.data_ptr(), weights.data_ptr() if weights is not None else None, y.data_ptr(), _ld(y),
              grad.data_ptr(), _ld(grad), _TYPE[y.dtype], dy.data_ptr() if dy is not None else None,
              max(width, 1), dw.data_ptr() if dw is not None else None)
        return dy, dw, None, None


def combine(y, plan, weights=None):
    """out [T, H]: out[t] = sum over j of weights[t, j] * y[plan.places[t, j]], summed in fp32 (differentiable).

    y [R, H] fp16 or bf16 in the plan's row order; weights [T, k] fp32, None for ones.  Dropped assignments add
    nothing.
    """
    if plan.places is None or plan.places.dim() != 2:
        raise ValueError("combine needs the plan's places, [tokens, k]")
    if y.dim() != 2:
        raise ValueError("y must be [rows, width]")
    if y.dtype not in _HALVES:
        raise TypeError(f"y must be float16 or bfloat16, got {y.dtype}")
    if not 1 <= plan.places.shape[1] <= _MAX_K:
        raise ValueError(f"k must lie in [1, {_MAX_K}]")
    _on_device(y, places=plan.places, weights=weights, offsets=plan.offsets)
    if weights is not None:
        if weights.dtype != torch.float32:
            raise TypeError(f"weights must be float32, got {weights.dtype}")
        if weights.shape != plan.places.shape:
            raise ValueError(f"weights must be {tuple(plan.places.shape)}, got {tuple(weights.shape)}")
        weights = weights.contiguous()
    places = _index(plan.places, "places")
    if not _tracked(y, weights):
        return _combine(_rows(y), places, weights, y.dtype)
    return _Combine.apply(y, weights, _index(plan.offsets, "offsets"), places)

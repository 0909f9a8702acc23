"""The experts' products of rows in their own type, and of rows and weights in 8 bits
(no counterparts in the reference, whose products are float64): segment_mm for the rows
that route_plan puts in order.

    weights, ids = topk_route(logits, k)
    plan = route_plan(ids, num_experts)
    y = combine_rows(expert_mm(dispatch_rows(x, plan), w, plan), weights, plan)

or, with the experts' weights kept in 8 bits,

    q = quantize_blocks(w)                                  # once
    rows = dispatch_rows(quantize_rows(x), plan)            # or of rms_norm(.., quantize=True)
    y = combine_rows(scaled_mm(rows, q, plan, dtype=x.dtype), weights, plan)

(rows brought to 8 bits in front of the dispatch are N, behind it N * k with the same bits:
32,768 bfloat16 rows of 4,096 to 2 of 32 experts in 767 us, the other way in 953). Sums are
float32 (float64 for float64 rows) and are rounded to the rows' type once.
"""

from __future__ import annotations

import torch

from .. import _lib
from ..base import DGLError
from . import _autograd
from . import quant as _quant
from .route import RoutePlan, _check_plan

__all__ = ["expert_mm", "scaled_mm"]


class _Groups:
    """The groups of a call's rows: their lengths on the GPU. A plan's are taken as they
    are, without waiting on the host; other lengths are checked there."""

    def __init__(self, plan, rows, groups, what):
        if isinstance(plan, RoutePlan):
            if plan.num_experts != groups:
                raise DGLError("{}: the plan is of {} experts, there are {} weights".format(
                    what, plan.num_experts, groups))
            if plan.num_rows * plan.k != rows:
                raise DGLError("{}: the plan is of {} entries, got {} rows".format(
                    what, plan.num_rows * plan.k, rows))
            self.plan, self.host = plan, None
            return
        self.plan, self.host = None, _lib.i64(plan)
        if self.host.ndim != 1 or self.host.size != groups:
            raise DGLError("{}: one length for each of {} weights wanted, got shape {}".format(
                what, groups, tuple(self.host.shape)))
        if groups:
            lo, hi = int(self.host.min()), int(self.host.max())
            # each length in [0, rows] before the sum: no int64 wrap-around
            total = int(self.host.sum()) if hi <= rows else rows + 1
            if lo < 0 or total > rows:
                raise DGLError("{}: lengths must be non-negative and sum to at most {}, got a "
                               "minimum of {} and a sum of {}".format(what, rows, lo, total))

    def on_device(self, what):
        if self.plan is not None:
            _check_plan(self.plan, what)
            _lib.used_here(self.plan._stream, self.plan.seglen)
            return self.plan.seglen
        return torch.from_numpy(self.host).to(_lib.device())


def expert_mm(value, weight, plan):
    r"""Each group of rows times its own matrix::

        y[i] = value[i] @ weight[g]      for row i of group g

    Parameters
    ----------
    value : (N, D1) array or tensor, the groups' rows one after the other
        (`dispatch_rows`); float16, bfloat16, float32 and float64 keep their type
    weight : (R, D1, D2) array or tensor of ``value``'s type. One whose last two axes
        are changed (``w.transpose(1, 2)`` of a contiguous (R, D2, D1)) is read as it lies
        in 16 bits, others are copied
    plan : the `RoutePlan` of the rows' N entries and R experts, whose lengths stay on
        the GPU (the call can be captured into a HIP graph), or the R lengths, which are
        checked on the host: non-negative, summing to at most N

    Returns
    -------
    (N, D2) products in ``value``'s type, zeros for rows behind the last group (entries
    of no expert). With torch tensors that require grad the result takes part in
    autograd; the weights' gradient is summed in a fixed order.
    """
    if _autograd.needs_grad(value, weight):
        return _autograd.ExpertMM.apply(value, weight, plan)
    y, _ = _expert_mm(value, weight, plan)
    return _lib.hand_back(y, _lib.caller_device(value, weight))


def _operands(value, weight, what):
    x, w = _lib.rows(value), _lib.rows(weight)
    if x.ndim != 2 or w.ndim != 3:
        raise DGLError("{} wants rows of shape (N, D1) and weights of shape (R, D1, D2), got {} "
                       "and {}".format(what, tuple(x.shape), tuple(w.shape)))
    if w.shape[1] != x.shape[1]:
        raise DGLError("{}: inner dimensions do not match: {} vs {}".format(
            what, x.shape[1], w.shape[1]))
    if x.dtype is not w.dtype:
        raise DGLError("{} wants rows and weights of one type, got {} and {}".format(
            what, x.dtype, w.dtype))
    return x, w


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


def _expert_mm(value, weight, plan):
    """(products, lengths) on the GPU."""
    x, w = _operands(value, weight, "expert_mm")
    (n, d1), (r, _, d2) = x.shape, w.shape
    groups = _Groups(plan, n, r, "expert_mm")
    dev = _lib.device()
    seglen = groups.on_device("expert_mm")
    x = _lib.rows_on_device(x, x.dtype)
    if x.dtype.itemsize > 2:
        return _wide_mm(x, _lib.rows_on_device(w, w.dtype), seglen), seglen
    w, transposed = _quant.matrices_on_device(w, w.dtype)
    y = torch.empty(n, d2, dtype=x.dtype, device=dev)
    _mm16(x, w, y, seglen, d1, r, d2, transposed)
    return y, seglen


def _mm16(x, w, y, seglen, d1, r, d2, transposed):
    L, n, code = _lib.lib(), x.shape[0], _lib.ROW_CODES[x.dtype]
    nbytes = L.mdgl_expert_mm_workspace_bytes(n, d1, r, d2, code)
    ws = _workspace(nbytes, x.device)
    _lib.check(L.mdgl_expert_mm(
        x.data_ptr(), w.data_ptr(), y.data_ptr(), seglen.data_ptr(), n, d1, r, d2, transposed,
        _lib.ptr(ws), nbytes, code, _lib.stream()), "expert_mm")


def _wide_mm(x, w, seglen):
    """float32 and float64 rows: segment_mm's kernels, which leave rows behind the last
    group as they are."""
    (n, d1), (r, _, d2) = x.shape, w.shape
    y = torch.zeros(n, d2, dtype=x.dtype, device=x.device)
    if n and r and d1 and d2:
        L, code = _lib.lib(), _lib.ROW_CODES[x.dtype]
        nbytes = L.mdgl_segment_mm_workspace_bytes(n, d1, d2, r, code)
        ws = _workspace(nbytes, x.device)
        _lib.check(L.mdgl_segment_mm(
            x.data_ptr(), w.data_ptr(), y.data_ptr(), seglen.data_ptr(), n, d1, r, d2,
            _lib.ptr(ws), nbytes, code, _lib.stream()), "segment_mm")
    return y


def _expert_mm_grad(value, weight, seglen, grad, need):
    """(dvalue, dweight) on the GPU, those that `need` wants."""
    x, w = _lib.rows(value), _lib.rows(weight)
    (n, d1), (r, _, d2) = x.shape, w.shape
    x = _lib.rows_on_device(x, x.dtype)
    g = _lib.rows_on_device(grad, x.dtype)
    if x.dtype.itemsize > 2:
        return _wide_mm_grad(x, _lib.rows_on_device(w, w.dtype), seglen, g, need)
    dx = dw = None
    if need[0]:
        w, transposed = _quant.matrices_on_device(w, w.dtype)
        dx = torch.empty_like(x)
        _mm16(g, w, dx, seglen, d2, r, d1, not transposed)
    if need[1]:
        dw = torch.empty(r, d1, d2, dtype=x.dtype, device=x.device)
        L, code = _lib.lib(), _lib.ROW_CODES[x.dtype]
        nbytes = L.mdgl_expert_mm_grad_workspace_bytes(n, d1, r, d2, code)
        ws = _workspace(nbytes, x.device)
        _lib.check(L.mdgl_expert_mm_grad(
            x.data_ptr(), g.data_ptr(), dw.data_ptr(), seglen.data_ptr(), n, d1, r, d2,
            _lib.ptr(ws), nbytes, code, _lib.stream()), "expert_mm_grad")
    return dx, dw


def _wide_mm_grad(x, w, seglen, g, need):
    (n, d1), (r, _, d2) = x.shape, w.shape
    dx = torch.zeros_like(x) if need[0] else None
    some = n and r and d1 and d2
    dw = (torch.empty_like if some else torch.zeros_like)(w) if need[1] else None
    if some:
        L, code = _lib.lib(), _lib.ROW_CODES[x.dtype]
        nbytes = L.mdgl_segment_mm_grad_workspace_bytes(n, d1, d2, r, code)
        ws = _workspace(nbytes, x.device)
        _lib.check(L.mdgl_segment_mm_grad(
            x.data_ptr(), w.data_ptr(), g.data_ptr(), seglen.data_ptr(), _lib.ptr(dx),
            _lib.ptr(dw), n, d1, r, d2, _lib.ptr(ws), nbytes, code, _lib.stream()),
            "segment_mm_grad")
    return dx, dw


_OUT_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def scaled_mm(value, weight, plan=None, dtype=None):
    r"""Products in 8 bits, with a scale for each block of 128::

        y[i, c] = sum_k (value.data * value.scale)[i, k] * (weight.data * weight.scale)[g, k, c]

    Parameters
    ----------
    value : `Quantized` rows (N, D1) (`quantize_rows`, `rms_norm`), or rows of float32,
        float16 or bfloat16, which are quantised first
    weight : `Quantized` matrices (`quantize_blocks`): (R, D1, D2), or one (D1, D2)
        for all rows. Memory with D1 innermost is read as it lies, other is copied
    plan : the `RoutePlan` of the rows' N entries and R experts, or the R lengths, as
        for `expert_mm`; None with one matrix
    dtype : of the products: float32, bfloat16 or float16. None: the rows', bfloat16 for
        `Quantized` ones

    Returns
    -------
    (N, D2) products, summed in float32 block by block, zeros for rows behind the last
    group. Within eight neighbouring k the matrix cores cut products off 13 binary
    places below the largest, so a sum is off by 7 * 2 ** -13 of these largest at most.
    Any finite scales may meet: a product of two below 2 ** -126 is rounded to a multiple
    of 2 ** -149, and where it is past float32's range a block's sum takes one after the
    other. It has no gradient (`expert_mm` has).
    """
    if not isinstance(weight, _quant.Quantized):
        raise DGLError("scaled_mm wants weights made by quantize_blocks")
    parts = (value if isinstance(value, _quant.Quantized) else (value,)) + tuple(weight)
    if _autograd.needs_grad(*parts):
        raise DGLError("scaled_mm has no gradient; expert_mm has")
    where = _lib.caller_device(*parts)
    if isinstance(value, _quant.Quantized):
        q, rows = value, None
        dtype = torch.bfloat16 if dtype is None else dtype
        _check_quantized(q, 1, "rows")
        shape = tuple(q.data.shape)
    else:
        q, rows = None, _quant._value(value, "scaled_mm")
        dtype = rows.dtype if dtype is None else dtype
        shape = tuple(rows.shape)
    if dtype not in _OUT_TYPES:
        raise DGLError("dtype must be one of {}, got {}".format(
            [str(t) for t in _OUT_TYPES], dtype))
    _check_quantized(weight, 2, "weights")
    w = weight.data
    if len(shape) != 2 or w.ndim not in (2, 3):
        raise DGLError("scaled_mm wants rows of shape (N, D1) and weights of shape (R, D1, D2) or "
                       "(D1, D2), got {} and {}".format(shape, tuple(w.shape)))
    n, d1 = shape
    r, d2 = (w.shape[0] if w.ndim == 3 else 1), w.shape[-1]
    if w.shape[-2] != d1:
        raise DGLError("scaled_mm: inner dimensions do not match: {} vs {}".format(
            d1, w.shape[-2]))
    if plan is None:
        if w.ndim == 3:
            raise DGLError("scaled_mm of several matrices wants a plan or lengths")
        groups = None
    else:
        groups = _Groups(plan, n, r, "scaled_mm")
    dev = _lib.device()
    seglen = None if groups is None else groups.on_device("scaled_mm")
    if q is None:
        q = _quant._quantize_rows(_lib.rows_on_device(rows, rows.dtype))
    data = _lib.rows_on_device(q.data, q.data.dtype)
    scale = _lib.rows_on_device(q.scale, torch.float32)
    w = _inner_last(w)
    ws_ = _lib.rows_on_device(weight.scale, torch.float32)
    if r == 0:  # and no lengths, which would be one group of all rows
        return _lib.hand_back(torch.zeros(n, d2, dtype=dtype, device=dev), where)
    y = torch.empty(n, d2, dtype=dtype, device=dev)
    L = _lib.lib()
    nbytes = L.mdgl_scaled_mm_workspace_bytes(n, d1, r, d2)
    ws = _workspace(nbytes, y.device)
    _lib.check(L.mdgl_scaled_mm(
        data.data_ptr(), scale.data_ptr(), w.data_ptr(), ws_.data_ptr(), y.data_ptr(),
        _lib.ptr(seglen), n, d1, r, d2, _lib.ptr(ws), nbytes, _lib.ROW_CODES[dtype],
        _lib.stream()), "scaled_mm")
    return _lib.hand_back(y, where)


def _check_quantized(q, axes, name):
    """Types and the scales' shape; `axes` of the last ones are in blocks."""
    data, scale = q
    if not isinstance(data, torch.Tensor) or not isinstance(scale, torch.Tensor) \
            or data.dtype is not torch.float8_e4m3fn or scale.dtype is not torch.float32:
        raise DGLError("quantized {} are float8_e4m3fn values with float32 scales".format(name))
    if data.ndim < axes:
        raise DGLError("quantized {} of shape {}".format(name, tuple(data.shape)))
    want = tuple(data.shape[:-axes]) + tuple(_quant.blocks(d) for d in data.shape[-axes:])
    if tuple(scale.shape) != want:
        raise DGLError("scales of the {} must have shape {}, got {}".format(
            name, want, tuple(scale.shape)))


def _inner_last(w):
    """The memory of (.., D1, D2) matrices with D1 innermost, on the current GPU."""
    t = w.transpose(-1, -2)
    if w.is_cuda and w.get_device() == _lib.current_device() and t.is_contiguous():
        return t
    return t.detach().to(_lib.device()).contiguous()

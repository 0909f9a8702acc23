"""Routing rows to experts, and the rows' way there and back (no counterpart in
the reference): what chooses the block of `gather_mm` / `segment_mm` for each
row, and puts the rows in that order.

    weights, ids = topk_route(logits, k)
    plan = route_plan(ids, num_experts)
    y = combine_rows(segment_mm(dispatch_rows(x, plan), w, plan.seglen), weights, plan)

Rows keep float32, float64, bfloat16 or float16; weights and sums are float32
(float64 for float64 rows). segment_mm takes 16-bit rows as float32 and returns
float32: `.to(x.dtype)` behind it keeps such a layer's rows in their type.
"""

from __future__ import annotations

import math

import torch

from .. import _lib
from ..base import DGLError
from . import _autograd

__all__ = ["RoutePlan", "topk_route", "route_plan", "dispatch_rows", "combine_rows"]

_SCORES = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORES = {"max": 0, "top2": 1}


def topk_route(logits, k, score="softmax", bias=None, num_groups=1, topk_groups=None,
               group_score="max", renormalize=True, scale=1.0):
    r"""Choose k experts for each row.

    Parameters
    ----------
    logits : (N, E) array or tensor, E at most 2048; -inf masks an expert
    k : experts a row, at most 32
    score : 'softmax' over the row's experts, or 'sigmoid' of each
    bias : (E,) finite, added to the scores for the choice only (to balance the
        experts' load); without it the logits' order decides
    num_groups : the experts fall into this many groups of neighbours (at most 64)
    topk_groups : only experts of this many best groups are chosen (None: all)
    group_score : a group's rank: its 'max' score, or the sum of its best two
        scores ('top2'), with the bias
    renormalize : divide a row's weights by their sum
    scale : factor of the weights

    Returns
    -------
    ``(weights, ids)``, both (N, k), best first, the lowest index among equals;
    ids are int64. Scores that differ by less than float32 shows are compared in
    float64. An expert masked by -inf is chosen only when nothing else is left and
    weighs 0; a NaN ranks with the masked and makes the weights it enters NaN. With
    torch logits that require grad the weights take part in autograd; `bias` gets no
    gradient.
    """
    if _autograd.needs_grad(logits):
        return _autograd.TopkRoute.apply(logits, k, score, bias, num_groups, topk_groups,
                                         group_score, renormalize, scale)
    w, ids = _topk_route(logits, k, score, bias, num_groups, topk_groups, group_score,
                         renormalize, scale)
    where = _lib.caller_device(logits)
    return _lib.hand_back(w, where), _lib.hand_back(ids, where)


def _topk_route(logits, k, score, bias, num_groups, topk_groups, group_score, renormalize, scale):
    """(weights, ids) on the GPU."""
    x = _lib.rows(logits)
    if x.ndim != 2:
        raise DGLError("topk_route wants logits of shape (N, E), got {}".format(tuple(x.shape)))
    if score not in _SCORES:
        raise DGLError("score must be one of {}, got {!r}".format(sorted(_SCORES), score))
    if group_score not in _GROUP_SCORES:
        raise DGLError("group_score must be one of {}, got {!r}".format(sorted(_GROUP_SCORES),
                                                                        group_score))
    n, e = x.shape
    xt = x.dtype
    st = _lib.state_dtype(xt)
    b = None if bias is None else _lib.rows(bias)
    if b is not None and tuple(b.shape) != (e,):
        raise DGLError("bias must have shape {}, got {}".format((e,), tuple(b.shape)))
    scale = float(scale)
    if not math.isfinite(scale):
        raise DGLError("scale must be finite, got {}".format(scale))
    dev = _lib.device()
    x = _lib.rows_on_device(x, xt)
    b = None if b is None else _lib.rows_on_device(b, st)
    k, num_groups = int(k), int(num_groups)
    topk_groups = num_groups if topk_groups is None else int(topk_groups)
    cols = min(max(k, 0), e)  # other k are refused below
    w = torch.empty(n, cols, dtype=st, device=dev)
    ids = torch.empty(n, cols, dtype=torch.int64, device=dev)
    _lib.check(_lib.lib().mdgl_topk_route(
        x.data_ptr(), _lib.ptr(b), w.data_ptr(), ids.data_ptr(), n, e, k, _SCORES[score],
        num_groups, topk_groups, _GROUP_SCORES[group_score], bool(renormalize), scale,
        _lib.ROW_CODES[xt], _lib.stream()), "topk_route")
    return w, ids


def _topk_route_grad(logits, ids, grad, score, renormalize, scale):
    x = _lib.rows(logits)
    n, e = x.shape
    xt = x.dtype
    x = _lib.rows_on_device(x, xt)
    g = _lib.rows_on_device(grad, _lib.state_dtype(xt))
    if ids.device != x.device:
        ids = ids.to(x.device)
    dx = torch.empty_like(x)
    _lib.check(_lib.lib().mdgl_topk_route_grad(
        x.data_ptr(), ids.data_ptr(), g.data_ptr(), dx.data_ptr(), n, e, ids.shape[1],
        _SCORES[score], bool(renormalize), float(scale), _lib.ROW_CODES[xt], _lib.stream()),
        "topk_route_grad")
    return dx


class RoutePlan:
    """Rows' entries in the order of their experts, on the GPU (`route_plan`).

    seglen : (E,) int64, entries of each expert: `segment_mm`'s lengths
    order : (N * k,) int32, the entry (row * k + choice) at each place
    slot : (N, k) int32, each entry's place; the complement (~) of it for an entry
        of no expert (these come last)
    """

    def __init__(self, ids, num_experts):
        on_gpu = isinstance(ids, torch.Tensor) and ids.device.type == "cuda"
        num_experts = int(num_experts)
        flat = _lib.i64_device(ids) if on_gpu else _lib.i64(ids)
        if flat.ndim not in (1, 2):
            raise DGLError("route_plan wants ids of shape (N, k) or (N,), got {}".format(
                tuple(flat.shape)))
        if not on_gpu:
            flat = torch.from_numpy(flat).to(_lib.device())
        L = _lib.lib()
        self.num_rows = flat.shape[0]
        self.k = flat.shape[1] if flat.ndim == 2 else 1
        self.num_experts = num_experts
        self.device_index, self._stream = _lib.current_device(), _lib.stream()
        m = flat.numel()
        dev = flat.device
        nbytes = L.mdgl_route_plan_workspace_bytes(m, num_experts)
        if nbytes < 0:  # refused before anything of that size is allocated
            _lib.check(L.mdgl_route_plan(None, m, num_experts, None, None, None, None, 0,
                                         _lib.stream()), "route_plan")
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes > 0 else None
        self.seglen = torch.empty(num_experts, dtype=torch.int64, device=dev)
        self.order = torch.empty(m, dtype=torch.int32, device=dev)
        self.slot = torch.empty(self.num_rows, self.k, dtype=torch.int32, device=dev)
        _lib.check(L.mdgl_route_plan(
            flat.data_ptr(), m, num_experts, self.seglen.data_ptr(), self.order.data_ptr(),
            self.slot.data_ptr(), _lib.ptr(ws), nbytes, _lib.stream()), "route_plan")


def route_plan(ids, num_experts) -> RoutePlan:
    """The order that puts each expert's rows together.

    Parameters
    ----------
    ids : (N, k) or (N,) integers, the experts of each row (`topk_route`'s); an id
        outside [0, num_experts) belongs to no expert (a padded row, an expert held
        elsewhere): `dispatch_rows` gives its entry zeros behind all others,
        `combine_rows` leaves it out
    num_experts : at most 2048

    Returns
    -------
    A `RoutePlan`. Its making does not wait on the host, and can be captured into
    a HIP graph when the ids are an int64 GPU tensor.
    """
    return RoutePlan(ids, num_experts)


def _check_plan(plan, what):
    if not isinstance(plan, RoutePlan):
        raise DGLError("{} wants a plan made by route_plan".format(what))
    if plan.device_index != _lib.current_device():
        raise DGLError("the plan lies on GPU {}, the current one is {}".format(
            plan.device_index, _lib.current_device()))
    _lib.used_here(plan._stream, plan.slot)


def dispatch_rows(value, plan):
    """Rows copied to their experts' places.

    Parameters
    ----------
    value : (N, ...) array or tensor
    plan : the `RoutePlan` of the N rows

    Returns
    -------
    (N * k, ...) rows in the experts' order, for `segment_mm` with
    ``plan.seglen``; zeros for entries of no expert. With a torch tensor that
    requires grad the result takes part in autograd.
    """
    if _autograd.needs_grad(value):
        return _autograd.DispatchRows.apply(value, plan)
    return _lib.hand_back(_dispatch_rows(value, plan), _lib.caller_device(value))


def _dispatch_rows(value, plan):
    x = _lib.rows(value)
    if x.ndim < 1:
        raise DGLError("dispatch_rows wants rows, got a value without axes")
    _lib.device()
    _check_plan(plan, "dispatch_rows")
    n, k, shape = plan.num_rows, plan.k, x.shape
    if shape[0] != n:
        raise DGLError("dispatch_rows: the plan is of {} rows, got {}".format(n, shape[0]))
    x = _lib.rows_on_device(x, x.dtype)
    out = torch.empty((n * k,) + tuple(shape[1:]), dtype=x.dtype, device=x.device)
    _lib.check(_lib.lib().mdgl_dispatch_rows(
        x.data_ptr(), plan.slot.data_ptr(), out.data_ptr(), n, k, math.prod(shape[1:]),
        _lib.ROW_CODES[x.dtype], _lib.stream()), "dispatch_rows")
    return out


def _sum_rows(x, weights, plan):
    """(N, ...) sums of the plan's entries of the contiguous GPU rows `x`."""
    n, k, d = plan.num_rows, plan.k, math.prod(x.shape[1:])
    out = torch.empty((n,) + tuple(x.shape[1:]), dtype=x.dtype, device=x.device)
    _lib.check(_lib.lib().mdgl_combine_rows(
        x.data_ptr(), plan.slot.data_ptr(), _lib.ptr(weights), out.data_ptr(), n, k, d,
        _lib.ROW_CODES[x.dtype], _lib.stream()), "combine_rows")
    return out


def combine_rows(value, weights, plan):
    """The experts' rows brought back: each row's weighted sum of its entries.

    Parameters
    ----------
    value : (N * k, ...) rows in the experts' order
    weights : (N, k) factor of each entry (`topk_route`'s)
    plan : the `RoutePlan` of the N rows

    Returns
    -------
    (N, ...) sums in the type of ``value``, added in float32 (float64) in the
    order of the choices. With torch tensors that require grad the result takes
    part in autograd.
    """
    if _autograd.needs_grad(value, weights):
        return _autograd.CombineRows.apply(value, weights, plan)
    return _lib.hand_back(_combine_rows(value, weights, plan),
                          _lib.caller_device(value, weights))


def _combine_operands(value, weights, plan):
    x, w = _lib.rows(value), _lib.rows(weights)
    if x.ndim < 1:
        raise DGLError("combine_rows wants rows, got a value without axes")
    _lib.device()
    _check_plan(plan, "combine_rows")
    n, k = plan.num_rows, plan.k
    if x.shape[0] != n * k:
        raise DGLError("combine_rows: the plan is of {} entries, got {} rows".format(
            n * k, x.shape[0]))
    if tuple(w.shape) != (n, k) and not (k == 1 and tuple(w.shape) == (n,)):
        raise DGLError("weights must have shape {}, got {}".format((n, k), tuple(w.shape)))
    return _lib.rows_on_device(x, x.dtype), _lib.rows_on_device(w, _lib.state_dtype(x.dtype))


def _combine_rows(value, weights, plan):
    x, w = _combine_operands(value, weights, plan)
    return _sum_rows(x, w, plan)


def _combine_rows_grad(value, weights, plan, grad, need):
    """(dvalue, dweights) on the GPU, those that `need` wants."""
    x, w = _combine_operands(value, weights, plan)
    n, k, d = plan.num_rows, plan.k, math.prod(x.shape[1:])
    g = _lib.rows_on_device(grad, x.dtype)
    dx = torch.empty_like(x) if need[0] else None
    # without columns the kernel writes nothing
    dw = (torch.empty_like if d else torch.zeros_like)(w) if need[1] else None
    _lib.check(_lib.lib().mdgl_combine_rows_grad(
        x.data_ptr(), plan.slot.data_ptr(), w.data_ptr(), g.data_ptr(), _lib.ptr(dx), _lib.ptr(dw),
        n, k, d, _lib.ROW_CODES[x.dtype], _lib.stream()), "combine_rows_grad")
    return dx, dw

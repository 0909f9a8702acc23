"""Routing rows to experts, and the rows' way there and back (no counterpart in
the reference): what chooses the block of `gather_mm` / `segment_mm` for each
row, and puts the rows in that order.

    weights, ids = topk_route(logits, k)
    plan = route_plan(ids, num_experts)
    y = combine_rows(segment_mm(dispatch_rows(x, plan), w, plan.seglen), weights, plan)

Rows keep float32, float64, bfloat16 or float16; weights and sums are float32
(float64 for float64 rows).
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
    bias : (E,) added to the scores for the choice only (to balance the experts'
        load); without it the logits' order decides
    num_groups : the experts fall into this many groups of neighbours (at most 64)
    topk_groups : only experts of this many best groups are chosen (None: all)
    group_score : a group's rank: its 'max' score, or its best two's sum ('top2'),
        with the bias
    renormalize : divide a row's weights by their sum
    scale : factor of the weights

    Returns
    -------
    ``(weights, ids)``, both (N, k), best first, the lowest index among equals;
    ids are int64. Scores that differ by less than float32 shows are compared in
    float64. An expert masked by -inf is chosen only when nothing else is left and
    weighs 0. With torch logits that require grad the weights take part in
    autograd; `bias` gets no gradient.
    """
    if _autograd.needs_grad(logits):
        return _autograd.TopkRoute.apply(logits, k, score, bias, num_groups, topk_groups,
                                         group_score, renormalize, scale)
    w, ids, back = _topk_route(logits, k, score, bias, num_groups, topk_groups, group_score,
                               renormalize, scale)
    return back(w), back(ids)


def _topk_route(logits, k, score, bias, num_groups, topk_groups, group_score, renormalize, scale):
    """(weights, ids, back): GPU tensors and the function that gives a result back
    in the caller's container."""
    X = _lib.rows(logits)
    if X.ndim != 2:
        raise DGLError("topk_route wants logits of shape (N, E), got {}".format(X.shape))
    for name, value, table in (("score", score, _SCORES),
                               ("group_score", group_score, _GROUP_SCORES)):
        if value not in table:
            raise DGLError("{} must be one of {}, got {!r}".format(name, sorted(table), value))
    n, e = X.shape
    st = _lib.state_dtype(X.dtype)
    B = None if bias is None else _lib.rows(bias)
    if B is not None and B.shape != (e,):
        raise DGLError("bias must have shape {}, got {}".format((e,), B.shape))
    scale = float(scale)
    if not math.isfinite(scale):
        raise DGLError("scale must be finite, got {}".format(scale))
    dev = _lib.device()
    x = _lib.rows_on_device(X, X.dtype)
    b = None if B is None else _lib.rows_on_device(B, st)
    k, num_groups = int(k), int(num_groups)
    topk_groups = num_groups if topk_groups is None else int(topk_groups)
    w = torch.empty(n, max(k, 0), dtype=st, device=dev)
    ids = torch.empty(n, max(k, 0), dtype=torch.int64, device=dev)
    _lib.check(_lib.lib().mdgl_topk_route(
        x.data_ptr(), _lib.ptr(b), w.data_ptr(), ids.data_ptr(), n, e, k, _SCORES[score],
        num_groups, topk_groups, _GROUP_SCORES[group_score], bool(renormalize), scale,
        _lib.ROW_CODES[X.dtype], _lib.stream()), "topk_route")
    return w, ids, lambda t: _lib.give_back(t, X.is_torch, X.device)


def _topk_route_grad(logits, ids, grad, score, renormalize, scale):
    X = _lib.rows(logits)
    n, e = X.shape
    dev = _lib.device()
    x = _lib.rows_on_device(X, X.dtype)
    g = grad.to(device=dev, dtype=_lib.state_dtype(X.dtype)).contiguous()
    dx = torch.empty(n, e, dtype=X.dtype, device=dev)
    _lib.check(_lib.lib().mdgl_topk_route_grad(
        x.data_ptr(), ids.data_ptr(), g.data_ptr(), dx.data_ptr(), n, e, ids.shape[1],
        _SCORES[score], bool(renormalize), float(scale), _lib.ROW_CODES[X.dtype], _lib.stream()),
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
        self.device_index = _lib.current_device()
        m = flat.numel()
        dev = flat.device
        nbytes = L.mdgl_route_plan_workspace_bytes(m, num_experts)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes > 0 else None
        self.seglen = torch.empty(max(num_experts, 0), dtype=torch.int64, device=dev)
        self.order = torch.empty(m, dtype=torch.int32, device=dev)
        self.slot = torch.empty(self.num_rows, self.k, dtype=torch.int32, device=dev)
        _lib.check(L.mdgl_route_plan(
            flat.data_ptr(), m, num_experts, self.seglen.data_ptr(), self.order.data_ptr(),
            self.slot.data_ptr(), _lib.ptr(ws), max(nbytes, 0), _lib.stream()), "route_plan")


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


def _check_plan(plan, what, rows, want):
    if not isinstance(plan, RoutePlan):
        raise DGLError("{} wants a plan made by route_plan".format(what))
    if rows != want:
        raise DGLError("{}: the plan is of {} rows, got {}".format(what, want, rows))
    if plan.device_index != _lib.current_device():
        raise DGLError("the plan lies on GPU {}, the current one is {}".format(
            plan.device_index, _lib.current_device()))


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
    out, back = _dispatch_rows(value, plan)
    return back(out)


def _dispatch_rows(value, plan):
    X = _lib.rows(value)
    if X.ndim < 1:
        raise DGLError("dispatch_rows wants rows, got a value without axes")
    _check_plan(plan, "dispatch_rows", X.shape[0], plan.num_rows if isinstance(
        plan, RoutePlan) else None)
    x = _lib.rows_on_device(X, X.dtype)
    n, k, d = plan.num_rows, plan.k, int(math.prod(X.shape[1:]))
    out = torch.empty((n * k,) + X.shape[1:], dtype=X.dtype, device=x.device)
    _lib.check(_lib.lib().mdgl_dispatch_rows(
        x.data_ptr(), plan.slot.data_ptr(), out.data_ptr(), n, k, d, _lib.ROW_CODES[X.dtype],
        _lib.stream()), "dispatch_rows")
    return out, lambda t: _lib.give_back(t, X.is_torch, X.device)


def _sum_rows(x, weights, plan):
    """(N, ...) sums of the plan's entries of the contiguous GPU rows `x`."""
    n, k, d = plan.num_rows, plan.k, int(math.prod(x.shape[1:]))
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
    out, back = _combine_rows(value, weights, plan)
    return back(out)


def _combine_operands(value, weights, plan):
    X, W = _lib.rows(value), _lib.rows(weights)
    if X.ndim < 1:
        raise DGLError("combine_rows wants rows, got a value without axes")
    _check_plan(plan, "combine_rows", X.shape[0], plan.num_rows * plan.k if isinstance(
        plan, RoutePlan) else None)
    if W.shape != (plan.num_rows, plan.k) and not (plan.k == 1 and W.shape == (plan.num_rows,)):
        raise DGLError("weights must have shape {}, got {}".format((plan.num_rows, plan.k),
                                                                   W.shape))
    return X, W, _lib.rows_on_device(X, X.dtype), \
        _lib.rows_on_device(W, _lib.state_dtype(X.dtype))


def _combine_rows(value, weights, plan):
    X, W, x, w = _combine_operands(value, weights, plan)
    as_torch, where = _lib.wants_torch(X, W), _lib.out_device(X, W)
    return _sum_rows(x, w, plan), lambda t: _lib.give_back(t, as_torch, where)


def _combine_rows_grad(value, weights, plan, grad, need):
    """(dvalue, dweights) on the GPU, those that `need` wants."""
    X, W, x, w = _combine_operands(value, weights, plan)
    n, k, d = plan.num_rows, plan.k, int(math.prod(X.shape[1:]))
    g = grad.to(device=x.device, dtype=X.dtype).contiguous()
    dx = torch.empty_like(x) if need[0] else None
    # without columns the kernel writes nothing
    dw = (torch.empty_like if d else torch.zeros_like)(w) if need[1] else None
    _lib.check(_lib.lib().mdgl_combine_rows_grad(
        x.data_ptr(), plan.slot.data_ptr(), w.data_ptr(), g.data_ptr(), _lib.ptr(dx), _lib.ptr(dw),
        n, k, d, _lib.ROW_CODES[X.dtype], _lib.stream()), "combine_rows_grad")
    return dx, dw

"""Layer norm (no counterpart in the reference): the normalisation of feature
rows in front of a layer, beside edge_softmax and segment_softmax.
"""

from __future__ import annotations

import torch

from .. import _lib
from ..base import DGLError
from . import _autograd

__all__ = ["layer_norm"]


def layer_norm(value, weight=None, bias=None, eps=1e-5):
    r"""Normalise each row over the last axis::

        y = (value - mean) / sqrt(var + eps) * weight + bias

    with ``var`` the mean of ``(value - mean) ** 2``.

    Parameters
    ----------
    value : (..., D) array or tensor; float32, float64, float16 and bfloat16
        keep their type, with the sums in float32 (float64 for float64)
    weight, bias : (D,) arrays or tensors, or None for 1 and 0; in the type of
        ``value`` or, beside 16-bit values, in float32 (float64 ones make the rows
        float64, too)
    eps : added to the variance, >= 0

    Returns
    -------
    The normalised rows, of ``value``'s shape and type. With torch tensors that
    require grad the result takes part in autograd; the weights' gradients are
    summed over the rows in a fixed order.
    """
    if _autograd.needs_grad(value, weight, bias):
        return _autograd.LayerNorm.apply(value, weight, bias, eps)
    y, _ = _layer_norm(value, weight, bias, eps, False)
    return _lib.hand_back(y, _lib.caller_device(value, weight, bias))


def _operands(value, weight, bias):
    """The operands and the types (rows, weights) of a call, checked."""
    x = _lib.rows(value)
    w = None if weight is None else _lib.rows(weight)
    b = None if bias is None else _lib.rows(bias)
    if x.ndim < 1:
        raise DGLError("layer_norm wants rows, got a value without axes")
    d = x.shape[-1]
    vt = wt = x.dtype
    for name, t in (("weight", w), ("bias", b)):
        if t is None:
            continue
        if t.ndim != 1 or t.shape[0] != d:
            raise DGLError("{} must have shape {}, got {}".format(name, (d,), tuple(t.shape)))
        if t.dtype is torch.float64:
            vt = wt = torch.float64
        elif t.dtype is not vt and wt is not torch.float64:
            wt = torch.float32
    return x, w, b, vt, wt, d


def _layer_norm(value, weight, bias, eps, want_stats):
    """(y, stats) on the GPU; stats: the rows' means, then their 1 / deviations."""
    x, w, b, vt, wt, d = _operands(value, weight, bias)
    eps = float(eps)
    if not eps >= 0.0:
        raise DGLError("eps must be >= 0, got {}".format(eps))
    _lib.device()
    x = _lib.rows_on_device(x, vt)
    w = None if w is None else _lib.rows_on_device(w, wt)
    b = None if b is None else _lib.rows_on_device(b, wt)
    n = x.numel() // d if d else 0
    y = torch.empty_like(x)
    stats = mean = rstd = None
    if want_stats:
        stats = torch.empty(2 * n, dtype=_lib.state_dtype(vt), device=x.device)
        mean, rstd = _stats_ptrs(stats)
    _lib.check(_lib.lib().mdgl_layer_norm(
        x.data_ptr(), _lib.ptr(w), _lib.ptr(b), y.data_ptr(), mean, rstd, n, d, eps,
        _lib.ROW_CODES[vt], _lib.ROW_CODES[wt], _lib.stream()), "layer_norm")
    return y, stats


def _stats_ptrs(stats):
    base = stats.data_ptr()
    return base, base + stats.numel() // 2 * stats.element_size()


def _layer_norm_grad(value, weight, bias, stats, grad, need):
    """(dvalue, dweight, dbias) on the GPU, those that `need` wants."""
    x, w, _, vt, wt, d = _operands(value, weight, bias)
    x = _lib.rows_on_device(x, vt)
    w = None if w is None else _lib.rows_on_device(w, wt)
    g = _lib.rows_on_device(grad, vt)
    dev = x.device
    n = x.numel() // d if d else 0
    dx = torch.empty_like(x) if need[0] else None
    # no rows: the kernels write nothing
    make = torch.empty if n else torch.zeros
    dw = make(d, dtype=wt, device=dev) if need[1] else None
    db = make(d, dtype=wt, device=dev) if need[2] else None
    L = _lib.lib()
    code = _lib.ROW_CODES[vt]
    ws, nbytes = None, 0
    if need[1] or need[2]:
        nbytes = L.mdgl_layer_norm_grad_workspace_bytes(n, d, code)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes > 0 else None
    _lib.check(L.mdgl_layer_norm_grad(
        x.data_ptr(), _lib.ptr(w), *_stats_ptrs(stats), g.data_ptr(), _lib.ptr(dx), _lib.ptr(dw),
        _lib.ptr(db), n, d, _lib.ptr(ws), nbytes, code, _lib.ROW_CODES[wt], _lib.stream()),
        "layer_norm_grad")
    return dx, dw, db

"""Layer norm and root-mean-square norm (no counterparts in the reference): the
normalisation of feature rows in front of a layer, beside edge_softmax and
segment_softmax.
"""

from __future__ import annotations

import torch

from .. import _lib
from ..base import DGLError
from . import _autograd
from . import quant as _quant

__all__ = ["layer_norm", "rms_norm"]


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


def rms_norm(value, weight=None, residual=None, eps=1e-6, quantize=False):
    r"""Normalise each row over the last axis by its root mean square, after a
    residual's addition::

        total = value + residual
        y = total / sqrt(mean(total ** 2) + eps) * weight

    Parameters
    ----------
    value : (..., D) array or tensor; float32, float64, float16 and bfloat16
        keep their type, with the sums in float32 (float64 for float64)
    weight : (D,) array or tensor, or None for 1; in the type of ``value`` or,
        beside 16-bit values, in float32 (float64 ones make the rows float64, too)
    residual : array or tensor of ``value``'s shape, or None for 0; types as for
        ``weight``, and ``total`` has its type
    eps : added to the mean square, >= 0
    quantize : return y as `Quantized` rows (`quantize_rows` of the unrounded y), for
        `scaled_mm`; not for float64, and without a gradient

    Returns
    -------
    y, of ``value``'s shape and type, and with a residual ``(y, total)``: total is the
    residual of the next layer. y is formed from the sum before it is rounded to
    total's type. With torch tensors that require grad the results take part in
    autograd; the weight's gradient is summed over the rows in a fixed order.
    """
    if _autograd.needs_grad(value, weight, residual):
        if quantize:
            raise DGLError("rms_norm has no gradient with quantize=True")
        y, total = _autograd.RmsNorm.apply(value, weight, residual, eps)
        return y if residual is None else (y, total)
    y, total, _, _ = _rms_norm(value, weight, residual, eps, bool(quantize), False)
    where = _lib.caller_device(value, weight, residual)
    y = _quant.hand_back(y, where) if quantize else _lib.hand_back(y, where)
    return y if residual is None else (y, _lib.hand_back(total, where))


def _rms_operands(value, weight, residual):
    """The operands and the types (rows, weight, residual) of a call, checked."""
    x, w, _, vt, wt, d = _operands(value, weight, None)
    r = None if residual is None else _lib.rows(residual)
    if r is not None and r.shape != x.shape:
        raise DGLError("residual must have shape {}, got {}".format(tuple(x.shape),
                                                                    tuple(r.shape)))
    if r is not None and r.dtype is torch.float64:
        vt = wt = torch.float64
    rt = vt if r is None or vt is torch.float64 or r.dtype is vt else torch.float32
    return x, w, r, vt, wt, rt, d


def _rms_norm(value, weight, residual, eps, quantize, want_stats):
    """(y, total, rstd) on the GPU and the types (rows, weight, residual)."""
    x, w, r, vt, wt, rt, d = _rms_operands(value, weight, residual)
    eps = float(eps)
    if not eps >= 0.0:
        raise DGLError("eps must be >= 0, got {}".format(eps))
    if quantize and vt is torch.float64:
        raise DGLError("quantize wants float32, float16 or bfloat16 rows, got float64")
    _lib.device()
    x = _lib.rows_on_device(x, vt)
    w = None if w is None else _lib.rows_on_device(w, wt)
    r = None if r is None else _lib.rows_on_device(r, rt)
    n = x.numel() // d if d else 0
    total = None if r is None else torch.empty_like(r)
    rstd = torch.empty(n, dtype=_lib.state_dtype(vt), device=x.device) if want_stats else None
    y, scale = _quant.empty_rows(x.shape, x.device) if quantize else (torch.empty_like(x), None)
    _lib.check(_lib.lib().mdgl_rms_norm(
        x.data_ptr(), _lib.ptr(r), _lib.ptr(w), y.data_ptr(), _lib.ptr(scale), _lib.ptr(total),
        _lib.ptr(rstd), n, d, eps, _lib.ROW_CODES[vt], _lib.ROW_CODES[wt], _lib.ROW_CODES[rt],
        _lib.stream()), "rms_norm")
    y = _quant.Quantized(y, scale) if quantize else y
    return y, total, rstd, (vt, wt, rt)


def _rms_norm_grad(total, residual, weight, rstd, grad, grad_total, vt, wt, rt, need):
    """(dvalue, dweight, dresidual) on the GPU, those that `need` wants, of rows that are
    `total` or, with a residual, the sum of both. One tensor serves both rows' gradients
    where they have one type."""
    t = _lib.rows_on_device(_lib.rows(total), rt)
    r = None if residual is None else _lib.rows_on_device(_lib.rows(residual), rt)
    gt = None if grad_total is None else _lib.rows_on_device(grad_total, rt)
    need_x, need_w, need_r = need
    if grad is None:  # y was not used: the sum's gradient alone
        dw = torch.zeros(t.shape[-1], dtype=wt, device=t.device) if need_w else None
        return gt.to(vt) if need_x else None, dw, gt if need_r else None
    w = None if weight is None else _lib.rows_on_device(_lib.rows(weight), wt)
    g = _lib.rows_on_device(grad, vt)
    d = t.shape[-1]
    n = t.numel() // d if d else 0
    one = rt is vt
    dx = torch.empty_like(g) if need_x or (need_r and one) else None
    dr = torch.empty_like(t) if need_r and not one else None
    # no rows: the kernels write nothing
    dw = (torch.empty if n else torch.zeros)(d, dtype=wt, device=t.device) if need_w else None
    L = _lib.lib()
    code = _lib.ROW_CODES[vt]
    ws, nbytes = None, 0
    if need_w:
        nbytes = L.mdgl_rms_norm_grad_workspace_bytes(n, d, code)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=t.device) if nbytes > 0 else None
    _lib.check(L.mdgl_rms_norm_grad(
        t.data_ptr(), _lib.ptr(r), _lib.ptr(w), rstd.data_ptr(), g.data_ptr(), _lib.ptr(gt),
        _lib.ptr(dx), _lib.ptr(dr), _lib.ptr(dw), n, d, _lib.ptr(ws), nbytes, code, _lib.ROW_CODES[wt],
        _lib.ROW_CODES[rt], _lib.stream()), "rms_norm_grad")
    return dx if need_x else None, dw, (dx if one else dr) if need_r else None

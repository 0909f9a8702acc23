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
        ``value`` or, beside 16-bit values, in float32
    eps : added to the variance, >= 0

    Returns
    -------
    The normalised rows, of ``value``'s shape and type. With torch tensors that
    require grad the result takes part in autograd; the weights' gradients are
    summed over the rows in a fixed order.
    """
    if _autograd.needs_grad(value, weight, bias):
        return _autograd.LayerNorm.apply(value, weight, bias, eps)
    y, _, _, back = _layer_norm(value, weight, bias, eps, False)
    return back(y)


def _operands(value, weight, bias):
    """Validated operands and the GPU types (rows, weights) of a call."""
    V = _lib.rows(value)
    W, B = (None if x is None else _lib.rows(x) for x in (weight, bias))
    if V.ndim < 1:
        raise DGLError("layer_norm wants rows, got a value without axes")
    d = V.shape[-1]
    for name, x in (("weight", W), ("bias", B)):
        if x is not None and x.shape != (d,):
            raise DGLError("{} must have shape {}, got {}".format(name, (d,), x.shape))
    given = {x.dtype for x in (W, B) if x is not None}
    vt = torch.float64 if torch.float64 in given else V.dtype
    wt = vt if given <= {vt} or vt == torch.float64 else torch.float32
    return V, W, B, vt, wt


def _layer_norm(value, weight, bias, eps, want_stats):
    """(y, mean, rstd, back): GPU tensors and the function that gives a result
    back in the caller's container."""
    V, W, B, vt, wt = _operands(value, weight, bias)
    eps = float(eps)
    if not eps >= 0.0:
        raise DGLError("eps must be >= 0, got {}".format(eps))
    d = V.shape[-1]
    dev = _lib.device()
    x = _lib.rows_on_device(V, vt)
    n = x.numel() // d if d else 0
    w, b = (None if t is None else _lib.rows_on_device(t, wt) for t in (W, B))
    y = torch.empty(V.shape, dtype=vt, device=dev)
    mean = rstd = None
    if want_stats:
        mean, rstd = torch.empty(2, n, dtype=_lib.state_dtype(vt), device=dev).unbind(0)
    _lib.check(_lib.lib().mdgl_layer_norm(
        x.data_ptr(), _lib.ptr(w), _lib.ptr(b), y.data_ptr(), _lib.ptr(mean), _lib.ptr(rstd), n, d,
        eps, _lib.ROW_CODES[vt], _lib.ROW_CODES[wt], _lib.stream()), "layer_norm")
    as_torch, where = _lib.wants_torch(V, W, B), _lib.out_device(V, W, B)
    return y, mean, rstd, lambda t: _lib.give_back(t, as_torch, where)


def _layer_norm_grad(value, weight, bias, mean, rstd, grad, need):
    """(dvalue, dweight, dbias) on the GPU, those that `need` wants."""
    V, W, B, vt, wt = _operands(value, weight, bias)
    d = V.shape[-1]
    dev = _lib.device()
    x = _lib.rows_on_device(V, vt)
    n = x.numel() // d if d else 0
    w = None if W is None else _lib.rows_on_device(W, wt)
    g = grad.to(device=dev, dtype=vt).contiguous()
    dx = torch.empty(V.shape, dtype=vt, device=dev) if need[0] else None
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
        x.data_ptr(), _lib.ptr(w), mean.data_ptr(), rstd.data_ptr(), g.data_ptr(), _lib.ptr(dx),
        _lib.ptr(dw), _lib.ptr(db), n, d, _lib.ptr(ws), nbytes, code, _lib.ROW_CODES[wt],
        _lib.stream()), "layer_norm_grad")
    return dx, dw, db

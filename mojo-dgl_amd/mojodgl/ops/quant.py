"""Values in 8 bits with scales (no counterpart in the reference): what rms_norm
can end in and scaled_mm multiplies.

A value is e4m3 (torch.float8_e4m3fn: 4 exponent bits, 3 mantissa bits, at most 448)
times the float32 scale of its block: 128 columns of a row, or 128 by 128 of a matrix.
"""

from __future__ import annotations

import math
from typing import NamedTuple

import torch

from .. import _lib
from ..base import DGLError
from . import _autograd

__all__ = ["Quantized", "quantize_rows", "quantize_blocks"]

BLOCK = 128


class Quantized(NamedTuple):
    """Values in 8 bits.

    data : float8_e4m3fn values; (..., D) rows, or (..., D1, D2) matrices whose memory
        has D1 innermost
    scale : float32 factors of their blocks; (..., ceil(D / 128)) or
        (..., ceil(D1 / 128), ceil(D2 / 128))
    """

    data: torch.Tensor
    scale: torch.Tensor


def blocks(d: int) -> int:
    """Blocks of 128 that d columns make."""
    return -(-d // BLOCK)


def hand_back(q: Quantized, where) -> Quantized:
    """`_lib.hand_back`, but left on the GPU for numpy callers: numpy has no e4m3."""
    return q if where is None else Quantized(*(_lib.hand_back(t, where) for t in q))


def _value(value, what):
    if isinstance(value, Quantized):
        raise DGLError("{} wants values, got quantized ones".format(what))
    if _autograd.needs_grad(value):
        raise DGLError("{} has no gradient".format(what))
    x = _lib.rows(value)
    if x.dtype is torch.float64:
        raise DGLError("{} takes float32, float16 or bfloat16, got float64".format(what))
    return x


def quantize_rows(value) -> Quantized:
    r"""Rows in 8 bits, a scale for each block of 128 columns::

        scale = max(max |value| / 448, 2 ** -126)
        data = value / scale, to the nearest e4m3 value (ties to even)

    Parameters
    ----------
    value : (..., D) array or tensor of float32, float16 or bfloat16

    Returns
    -------
    `Quantized` rows (GPU tensors for numpy rows). A NaN stays a NaN and leaves its
    block's scale alone; an infinity makes its block's scale infinite, and all the block
    NaN once multiplied back. It has no gradient.
    """
    x = _value(value, "quantize_rows")
    if x.ndim < 1:
        raise DGLError("quantize_rows wants rows, got a value without axes")
    _lib.device()
    x = _lib.rows_on_device(x, x.dtype)
    return hand_back(_quantize_rows(x), _lib.caller_device(value))


def _quantize_rows(x) -> Quantized:
    """Contiguous rows on the GPU."""
    d = x.shape[-1]
    n = x.numel() // d if d else 0
    q, scale = empty_rows(x.shape, x.device)
    _lib.check(_lib.lib().mdgl_quantize_rows(
        x.data_ptr(), q.data_ptr(), scale.data_ptr(), n, d, _lib.ROW_CODES[x.dtype],
        _lib.stream()), "quantize_rows")
    return Quantized(q, scale)


def empty_rows(shape, device) -> Quantized:
    data = torch.empty(tuple(shape), dtype=torch.float8_e4m3fn, device=device)
    scale = torch.empty(tuple(shape[:-1]) + (blocks(shape[-1]),), dtype=torch.float32,
                        device=device)
    return Quantized(data, scale)


def quantize_blocks(weight) -> Quantized:
    r"""Matrices in 8 bits, a scale for each block of 128 by 128 (as `quantize_rows`
    has one for 128 columns): the weights of `scaled_mm`.

    Parameters
    ----------
    weight : (..., D1, D2) array or tensor of float32, float16 or bfloat16

    Returns
    -------
    `Quantized` matrices, (..., D1, D2) with D1 innermost in memory, as the products
    read them. It has no gradient.
    """
    x = _value(weight, "quantize_blocks")
    if x.ndim < 2:
        raise DGLError("quantize_blocks wants matrices, got shape {}".format(tuple(x.shape)))
    _lib.device()
    x, transposed = matrices_on_device(x, x.dtype)
    d1, d2 = x.shape[-2:]
    lead = tuple(x.shape[:-2])
    data = torch.empty(lead + (d2, d1), dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(lead + (blocks(d1), blocks(d2)), dtype=torch.float32, device=x.device)
    _lib.check(_lib.lib().mdgl_quantize_blocks(
        x.data_ptr(), data.data_ptr(), scale.data_ptr(), math.prod(lead), d1, d2, transposed,
        _lib.ROW_CODES[x.dtype], _lib.stream()), "quantize_blocks")
    return hand_back(Quantized(data.transpose(-1, -2), scale), _lib.caller_device(weight))


def matrices_on_device(t, dtype):
    """(tensor, transposed): matrices of `dtype` on the current GPU whose memory is
    contiguous, as they are shaped or with the last two axes changed."""
    if t.dtype is dtype and t.is_cuda and t.get_device() == _lib.current_device() \
            and not t.is_contiguous() and t.transpose(-1, -2).is_contiguous():
        return t.detach(), True
    return _lib.rows_on_device(t, dtype), False

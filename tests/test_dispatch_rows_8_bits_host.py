"""Rows in 8 bits that require a gradient are refused by dispatch_rows, `Quantized` or not,
before any GPU work: their gradient would be a sum in 8 bits."""

import pytest
import torch

import mojodgl.ops as ops
from mojodgl import DGLError

F8 = torch.float8_e4m3fn


def test_rows_in_8_bits_have_no_gradient():
    x = torch.ones(4, 8).to(F8).requires_grad_()
    scale = torch.ones(4, 1)
    for bad in (x, ops.Quantized(x, scale),
                ops.Quantized(x.detach(), scale.clone().requires_grad_())):
        with pytest.raises(DGLError, match="no gradient"):
            ops.dispatch_rows(bad, None)

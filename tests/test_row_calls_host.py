"""Calls that are refused before any GPU work."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import mojodgl.ops as ops
from mojodgl import DGLError


def test_tangents_are_refused():
    """Forward mode has no kernels: a tangent is refused, never dropped."""
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.ones(4, 3), torch.ones(4, 3))
        y, w = torch.ones(4, 3), torch.ones(2, 3, 3)
        for call in (lambda: ops.layer_norm(x), lambda: ops.layer_norm(y, x[0]),
                     lambda: ops.segment_scan([4], y, x), lambda: ops.segment_scan([4], x, y),
                     lambda: ops.segment_scan([1, 3], y, y, x[:2]),
                     lambda: ops.segment_scan_step(y, y, x), lambda: ops.topk_route(x, 2),
                     lambda: ops.dispatch_rows(x, None), lambda: ops.combine_rows(y, x, None),
                     lambda: ops.segment_reduce([4], x), lambda: ops.segment_softmax([4], x),
                     lambda: ops.segment_mm(x, w, [2, 2]),
                     lambda: ops.gather_mm(x, w, idx_b=[0, 1, 0, 1])):
            with pytest.raises(DGLError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(DGLError, match="tangent"):
                call()
    with pytest.raises(DGLError, match="tangent"):
        torch.func.jvp(ops.layer_norm, (torch.ones(4, 3),), (torch.ones(4, 3),))

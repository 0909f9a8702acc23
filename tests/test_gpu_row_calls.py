"""Calls of the row operators beside others: what autograd saved and is written over."""

import pytest
import torch

import mojodgl.ops as ops

pytestmark = pytest.mark.gpu


def test_a_step_into_a_saved_state_is_seen_by_the_backward_pass():
    """`initial` is saved for the gates' gradient; a step that writes over it makes the
    backward pass raise, as torch's own in-place operations do."""
    gate = torch.rand(5, 4, device="cuda", requires_grad=True)
    value, state = torch.rand(5, 4, device="cuda"), torch.rand(2, 4, device="cuda")
    h = ops.segment_scan([2, 3], gate, value, state)
    version = state._version
    ops.segment_scan_step(value[:2], value[2:4], state, out=state)
    assert state._version == version + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    # into another tensor: the saved one is as it was
    out = torch.empty_like(state)
    h = ops.segment_scan([2, 3], gate, value, state)
    ops.segment_scan_step(value[:2], value[2:4], state, out=out)
    assert state._version == version + 1 and out._version == 1
    h.sum().backward()
    assert gate.grad is not None
    with torch.inference_mode():  # tensors without versions
        mine = torch.rand(2, 4, device="cuda")
        ops.segment_scan_step(mine, mine, mine.clone(), out=torch.empty_like(mine))

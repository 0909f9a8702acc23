"""Calls of the row operators without a GPU: refusals before any GPU work, and where a
backward pass runs."""

import contextlib
from types import SimpleNamespace

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import mojodgl.ops as ops
from mojodgl import DGLError, _lib
from mojodgl.ops import _autograd


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


def test_a_backward_pass_runs_where_its_forward_pass_ran(monkeypatch):
    """Autograd runs it on the results' GPU, which is the operands' and need not be the one
    that was current: the plan and the statistics lie there, and the kernels belong on
    that GPU's stream."""
    entered = []

    def note(kind):
        @contextlib.contextmanager
        def enter(what):
            entered.append((kind, what))
            yield
            entered.append((kind, None))
        return enter

    monkeypatch.setattr(torch.cuda, "device", note("device"))
    monkeypatch.setattr(torch.cuda, "stream", note("stream"))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: "queue 0")
    now = SimpleNamespace(gpu=0)
    monkeypatch.setattr(_lib, "current_device", lambda: now.gpu)
    run = _autograd._where_made(lambda ctx, a, b: entered.append((a, b)) or "grads")
    for where, later, want in ((torch.device("cuda", 0), 0, []),
                               (torch.device("cpu"), 0, []), (None, 0, []),
                               (torch.device("cpu"), 1, [("device", 0)]),
                               (torch.device("cuda", 1), 1, [("stream", "queue 0")])):
        ctx, now.gpu = SimpleNamespace(), 0
        _autograd._made_here(ctx, where)
        now.gpu = later
        assert run(ctx, 1, 2) == "grads"
        assert entered == want + [(1, 2)] + [(kind, None) for kind, _ in want]
        entered.clear()
    for name in ("SegmentScan", "LayerNorm", "TopkRoute", "DispatchRows", "CombineRows"):
        # once_differentiable around it, around the pass itself
        backward = getattr(_autograd, name).backward
        assert backward.__wrapped__.__code__ is run.__code__, name


def test_no_segments_at_all_is_nothing_to_do():
    """`has_empty` without a segment launches nothing."""
    lib, p = _lib.lib(), 4096  # an aligned address that is not read
    assert lib.mdgl_segment_scan(p, p, None, p, p, p, p, p, p, None, 0, 0, 16, 1, None, 0, 0, 0,
                                 None) == 0
    assert lib.mdgl_segment_scan_grad(p, p, None, p, p, None, p, p, p, p, p, p, p, 0, 0, 16, 1,
                                      None, 0, 0, 0, None) == 0

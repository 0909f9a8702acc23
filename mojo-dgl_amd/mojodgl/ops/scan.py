"""Gated linear recurrence over the rows of segments (no counterpart in the
reference): a sequence layer over packed, ragged sequences, beside
segment_reduce and segment_softmax.

Values keep float32, float64, bfloat16 or float16; states are float32
(float64 for float64 values).
"""

from __future__ import annotations

import math

import torch

from .. import _lib
from ..base import DGLError
from . import _autograd
from .segment import _Segments

__all__ = ["SegmentPlan", "segment_plan", "segment_scan", "segment_scan_step"]

MARK_ROWS = 16  # rows between the states kept for the backward pass


class SegmentPlan:
    """A batch's segments as the scan walks them, on the GPU: made once by
    `segment_plan` and used by every layer's scan of that batch.

    num_rows, num_segments : its rows and segments
    """

    def __init__(self, seglen, num_rows=None):
        if num_rows is None:
            on_gpu = isinstance(seglen, torch.Tensor) and seglen.device.type == "cuda"
            lengths = _lib.i64_device(seglen) if on_gpu else _lib.i64(seglen)
            num_rows = int(lengths.sum())
        num_rows = int(num_rows)
        if not 0 <= num_rows < 2 ** 31:
            raise DGLError("segment operators take fewer than 2**31 rows, got {}".format(num_rows))
        seg = _Segments(seglen, num_rows)  # raises for lengths that do not fit the rows
        dev = _lib.device()
        self.num_rows, self.num_segments = num_rows, seg.num
        self.has_empty = bool(seg.num) and seg.shortest == 0
        self.offsets = seg.device()
        self.device_index, self._stream = _lib.current_device(), _lib.stream()
        words = (num_rows + 63) // 64
        self.ids = torch.empty(num_rows, dtype=torch.int32, device=dev)
        self.starts = torch.empty(words, dtype=torch.int64, device=dev)
        self.ends = torch.empty(words, dtype=torch.int64, device=dev)
        _lib.check(_lib.lib().mdgl_segment_marks(
            self.offsets.data_ptr(), self.num_segments, num_rows, self.ids.data_ptr(),
            self.starts.data_ptr(), self.ends.data_ptr(), _lib.stream()), "segment_marks")
        _lib.settle()  # another stream that is given the plan reads it whole


def segment_plan(seglen, num_rows=None) -> SegmentPlan:
    """The layout of segments of `seglen` rows, to pass to `segment_scan` in
    place of the lengths.

    Its making waits on the host (the lengths are checked); the scans that take
    it do not, so they can be captured into a HIP graph.

    Parameters
    ----------
    seglen : lengths of the segments, non-negative, zeros allowed
    num_rows : their sum, checked when given
    """
    return SegmentPlan(seglen, num_rows)


def _types(value: torch.dtype, gate: torch.dtype):
    """(value, gate) types of a call: float64 when either is, else the value's
    type, with the gates in it or, beside 16-bit values, in float32."""
    if torch.float64 in (value, gate):
        return torch.float64, torch.float64
    return value, (value if gate == value else torch.float32)


def segment_scan(seglen, gate, value, initial=None, return_state=False):
    r"""Gated linear recurrence along each segment, per column::

        h[t] = gate[t] * h[t-1] + value[t]

    where ``h[-1]`` is the segment's row of ``initial``, or 0.

    Parameters
    ----------
    seglen : lengths of the segments, summing to N (zeros allowed), or the
        `SegmentPlan` made of them
    gate : (N, ...) array or tensor; with float16 / bfloat16 values it may be
        float32
    value : (N, ...) array or tensor of the same shape
    initial : (len(seglen), ...) states in front of the first rows
    return_state : also return each segment's state behind its last row
        (the initial state of an empty one)

    Returns
    -------
    ``h`` in the type of ``value`` (float64 beside a float64 gate), and with
    ``return_state`` the states, (len(seglen), ...) in float32 (float64 for float64
    ``h``), which the next
    call takes as ``initial``. With torch tensors that require grad the results
    take part in autograd. Products of the gates of a segment's neighbouring rows
    are formed: they must not overflow (gates in [-1, 1] never do), and where one is
    too small for the type an infinite state in front of it gives NaN, as behind a
    gate of 0.

    Examples
    --------
    >>> gate = np.full((5, 1), 0.5)
    >>> segment_scan([2, 0, 3], gate, np.ones((5, 1)))
    array([[1.  ],
           [1.5 ],
           [1.  ],
           [1.5 ],
           [1.75]])
    """
    if _autograd.needs_grad(gate, value, initial):
        h, last = _autograd.SegmentScan.apply(seglen, gate, value, initial, bool(return_state))
        return (h, last) if return_state else h
    h, last, _, _ = _scan(seglen, gate, value, initial, return_state, False)
    where = _lib.caller_device(value, gate, initial)
    h = _lib.hand_back(h, where)
    return (h, _lib.hand_back(last, where)) if return_state else h


def _scan(seglen, gate, value, initial, want_state, want_marks):
    """(h, last, marks, plan), the first three on the GPU."""
    g, v = _lib.rows(gate), _lib.rows(value)
    i = None if initial is None else _lib.rows(initial)
    shape = v.shape
    if v.ndim < 1 or g.shape != shape:
        raise DGLError("segment_scan wants a gate for every value, got shapes {} and {}".format(
            tuple(g.shape), tuple(shape)))
    n, d = shape[0], math.prod(shape[1:])
    plan = _plan_for(seglen, n)
    states = (plan.num_segments,) + tuple(shape[1:])
    if i is not None and tuple(i.shape) != states:
        raise DGLError("initial states of shape {} wanted, got {}".format(states, tuple(i.shape)))
    vt, gt = _types(v.dtype, g.dtype)
    st = _lib.state_dtype(vt)
    dev = _lib.device()
    g, v = _lib.rows_on_device(g, gt), _lib.rows_on_device(v, vt)
    i = None if i is None else _lib.rows_on_device(i, st)
    h = torch.empty_like(v)
    last = torch.empty(states, dtype=st, device=dev) if want_state else None
    marks = None
    if want_marks:
        marks = torch.empty((n + MARK_ROWS - 1) // MARK_ROWS, d, dtype=st, device=dev)
    L = _lib.lib()
    code = _lib.ROW_CODES[vt]
    nbytes = L.mdgl_segment_scan_workspace_bytes(n, d, code)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes > 0 else None
    _lib.check(L.mdgl_segment_scan(
        g.data_ptr(), v.data_ptr(), _lib.ptr(i), plan.offsets.data_ptr(), plan.ids.data_ptr(),
        plan.starts.data_ptr(), plan.ends.data_ptr(), h.data_ptr(), _lib.ptr(last),
        _lib.ptr(marks), plan.num_segments, n, d, plan.has_empty, _lib.ptr(ws), nbytes, code,
        _lib.ROW_CODES[gt], _lib.stream()), "segment_scan")
    return h, last, marks, plan


def _plan_for(seglen, n) -> SegmentPlan:
    if not isinstance(seglen, SegmentPlan):
        return SegmentPlan(seglen, n)
    if seglen.num_rows != n:
        raise DGLError("a plan of {} rows cannot lay out {}".format(seglen.num_rows, n))
    if seglen.device_index != _lib.current_device():
        raise DGLError("the plan lies on GPU {}, the current one is {}".format(
            seglen.device_index, _lib.current_device()))
    _lib.used_here(seglen._stream, seglen.offsets, seglen.ids, seglen.starts, seglen.ends)
    return seglen


def _scan_grad(plan, gate, value, initial, marks, grad, grad_last, need):
    """Gradients (GPU tensors or None) of gate, value and initial; `need` says
    which are wanted."""
    g, v = _lib.rows(gate), _lib.rows(value)
    vt, gt = _types(v.dtype, g.dtype)
    st = _lib.state_dtype(vt)
    dev = _lib.device()
    shape = tuple(v.shape)
    n, d = shape[0], math.prod(shape[1:])
    g, v = _lib.rows_on_device(g, gt), _lib.rows_on_device(v, vt)
    i = None if initial is None else _lib.rows_on_device(_lib.rows(initial), st)
    gh = torch.zeros(shape, dtype=vt, device=dev) if grad is None else \
        _lib.rows_on_device(grad, vt)
    gl = None if grad_last is None else _lib.rows_on_device(grad_last, st)
    dg = torch.empty(shape, dtype=gt, device=dev) if need[0] else None
    dv = torch.empty(shape, dtype=vt, device=dev) if need[1] else None
    di = None
    if need[2]:
        di = torch.empty((plan.num_segments,) + shape[1:], dtype=st, device=dev)
    L = _lib.lib()
    code = _lib.ROW_CODES[vt]
    nbytes = L.mdgl_segment_scan_workspace_bytes(n, d, code)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes > 0 else None
    _lib.check(L.mdgl_segment_scan_grad(
        g.data_ptr(), v.data_ptr(), _lib.ptr(i), marks.data_ptr(), gh.data_ptr(), _lib.ptr(gl),
        plan.offsets.data_ptr(), plan.ids.data_ptr(), plan.starts.data_ptr(),
        plan.ends.data_ptr(), _lib.ptr(dg), _lib.ptr(dv), _lib.ptr(di), plan.num_segments, n, d,
        plan.has_empty, _lib.ptr(ws), nbytes, code, _lib.ROW_CODES[gt],
        _lib.stream()), "segment_scan_grad")
    return dg, dv, di


def segment_scan_step(gate, value, state, out=None):
    """One row of every sequence: the recurrence of `segment_scan` continued by
    a row each, for answering.

    Parameters
    ----------
    gate, value : (S, ...) one row a sequence, types as in `segment_scan`
    state : (S, ...) the sequences' states, float32 (float64 for float64 values)
    out : tensor of the new states (a contiguous GPU tensor like the result's);
        it may be ``state`` itself, which is then updated in place (autograd counts
        it as torch's in-place operations)

    Returns
    -------
    ``(h, new_state)``: h in the type of ``value`` (float64 beside a float64 gate).
    It has no gradient (`segment_scan` has). One call takes fewer than 2**32 values.
    """
    if _autograd.needs_grad(gate, value, state):
        raise DGLError("segment_scan_step has no gradient; segment_scan has")
    g, v, s = _lib.rows(gate), _lib.rows(value), _lib.rows(state)
    if g.shape != v.shape or s.shape != v.shape:
        raise DGLError("segment_scan_step wants a gate, a value and a state of one shape, got "
                       "{}, {} and {}".format(*(tuple(t.shape) for t in (g, v, s))))
    vt, gt = _types(v.dtype, g.dtype)
    st = _lib.state_dtype(vt)
    _lib.device()
    where = _lib.caller_device(value, gate, state, out)
    if out is not None:
        if not isinstance(out, torch.Tensor) or not out.is_cuda or out.dtype != st \
                or out.shape != s.shape or not out.is_contiguous() \
                or out.get_device() != _lib.current_device():
            raise DGLError("out must be a contiguous {} tensor of shape {} on the current "
                           "GPU".format(st, tuple(s.shape)))
        if out.requires_grad and torch.is_grad_enabled():
            raise DGLError("out must not require grad")
    g, v, s = _lib.rows_on_device(g, gt), _lib.rows_on_device(v, vt), _lib.rows_on_device(s, st)
    h = torch.empty_like(v)
    if out is None:
        new = torch.empty_like(s)
    else:
        new = out
        for t in (g, v, s):
            if _overlap(new, t) and not (t is s and t.data_ptr() == new.data_ptr()):
                raise DGLError("out overlaps an operand it is not")
    _lib.check(_lib.lib().mdgl_segment_scan_step(
        g.data_ptr(), v.data_ptr(), s.data_ptr(), h.data_ptr(), new.data_ptr(), v.numel(),
        _lib.ROW_CODES[vt], _lib.ROW_CODES[gt], _lib.stream()), "segment_scan_step")
    if out is not None:
        # a backward pass that saved what was written over now raises
        torch.autograd.graph.increment_version(out)
    return _lib.hand_back(h, where), new if out is not None else _lib.hand_back(new, where)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory of two contiguous GPU tensors meets."""
    lo_a, lo_b = a.data_ptr(), b.data_ptr()
    return lo_a < lo_b + b.numel() * b.element_size() and \
        lo_b < lo_a + a.numel() * a.element_size()

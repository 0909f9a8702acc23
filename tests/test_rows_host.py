"""The operators over packed rows (layer norm, the segment scan, routing) without a
GPU: refusals of the Python layer before any GPU work, and of the C ABI before a
launch."""

import numpy as np
import pytest
import torch

import mojodgl as dgl
import mojodgl.nn.functional as nnf
import mojodgl.ops as ops
from mojodgl import DGLError, _lib

F32, F64, BF16, F16 = 0, 1, 2, 3
EINVAL, EWORKSPACE = -1, -2


def test_names():
    assert nnf.layer_norm is ops.layer_norm is dgl.layer_norm
    for name in ("segment_plan", "segment_scan", "segment_scan_step", "topk_route", "route_plan",
                 "dispatch_rows", "combine_rows", "SegmentPlan", "RoutePlan"):
        assert getattr(dgl, name) is getattr(ops, name) and getattr(ops, name).__doc__
        assert name in dgl.__all__


def test_layer_norm_refusals():
    x = np.zeros((3, 4), np.float32)
    for bad in (np.zeros(3), np.zeros((1, 4)), np.zeros(5, np.float32)):
        with pytest.raises(DGLError, match="weight"):
            ops.layer_norm(x, bad)
        with pytest.raises(DGLError, match="bias"):
            ops.layer_norm(torch.zeros(3, 4), None, torch.as_tensor(bad))
    with pytest.raises(DGLError, match="axes"):
        ops.layer_norm(np.float32(1.0))
    with pytest.raises(DGLError, match="complex"):
        ops.layer_norm(x.astype(np.complex64))
    for eps in (-1.0, float("nan")):
        with pytest.raises(DGLError, match="eps"):
            ops.layer_norm(x, eps=eps)


def test_scan_refusals():
    x = np.zeros((5, 2), np.float32)
    with pytest.raises(DGLError, match="gate for every value"):
        ops.segment_scan([5], x[:, :1], x)
    with pytest.raises(DGLError, match="gate for every value"):
        ops.segment_scan([1], np.float32(1), np.float32(1))
    for lens in ([4], [6], [-1, 6], [2, 2, 2]):
        with pytest.raises(DGLError, match="segment lengths"):
            ops.segment_scan(lens, x, x)
    with pytest.raises(DGLError, match="2\\*\\*31"):
        ops.segment_plan([2 ** 31])
    with pytest.raises(DGLError, match="one shape"):
        ops.segment_scan_step(x, x, x[:3])
    with pytest.raises(DGLError, match="no gradient"):
        ops.segment_scan_step(torch.zeros(2, 2, requires_grad=True), torch.zeros(2, 2),
                              torch.zeros(2, 2))


def test_route_refusals():
    x = np.zeros((3, 4), np.float32)
    with pytest.raises(DGLError, match="shape"):
        ops.topk_route(x[0], 1)
    with pytest.raises(DGLError, match="score must be one of"):
        ops.topk_route(x, 1, score="tanh")
    with pytest.raises(DGLError, match="group_score must be one of"):
        ops.topk_route(x, 1, group_score="mean")
    with pytest.raises(DGLError, match="bias"):
        ops.topk_route(x, 1, bias=np.zeros(3))
    for scale in (float("inf"), float("nan")):
        with pytest.raises(DGLError, match="scale"):
            ops.topk_route(x, 1, scale=scale)
    with pytest.raises(DGLError, match="ids of shape"):
        ops.route_plan(np.zeros((2, 2, 2), np.int64), 3)
    with pytest.raises(DGLError, match="whole numbers"):
        ops.route_plan(np.array([0.5]), 3)


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def err(lib):
    return lib.mdgl_last_error().decode()


P = 4096  # an aligned address that no refused call reads


def test_abi_segment_marks(lib):
    assert lib.mdgl_segment_marks(None, 0, 0, None, None, None, None) == 0
    assert lib.mdgl_segment_marks(P, -1, 5, P, P, P, None) == EINVAL
    assert lib.mdgl_segment_marks(P, 0, 5, P, P, P, None) == EINVAL and "segments" in err(lib)
    assert lib.mdgl_segment_marks(P, 1, 2 ** 31, P, P, P, None) == EINVAL
    assert lib.mdgl_segment_marks(P, 1, 5, P, None, P, None) == EINVAL and "null" in err(lib)


def test_abi_segment_scan(lib):
    need = lib.mdgl_segment_scan_workspace_bytes(1000, 16, F32)
    assert need > 0 and lib.mdgl_segment_scan_workspace_bytes(128, 16, F32) == 0
    assert lib.mdgl_segment_scan_workspace_bytes(1000, 16, 9) == -1
    assert lib.mdgl_segment_scan_workspace_bytes(0, 16, F32) == 0

    def scan(gate=P, value=P, off=P, ids=P, starts=P, ends=P, dst=P, last=None, segs=2, n=1000,
             d=16, empty=0, ws=P, nbytes=need, dt=F32, gdt=F32):
        return lib.mdgl_segment_scan(gate, value, None, off, ids, starts, ends, dst, last, None,
                                     segs, n, d, empty, ws, nbytes, dt, gdt, None)

    def grad(gate=P, value=P, marks=P, g=P, off=P, ids=P, starts=P, ends=P, dg=P, dv=P, di=None,
             segs=2, n=1000, d=16, empty=0, ws=P, nbytes=need, dt=F32, gdt=F32):
        return lib.mdgl_segment_scan_grad(gate, value, None, marks, g, None, off, ids, starts,
                                          ends, dg, dv, di, segs, n, d, empty, ws, nbytes, dt,
                                          gdt, None)

    for call in (scan, grad):
        assert call(n=0) == 0 and call(d=0) == 0
        for kw in (dict(dt=4), dict(dt=-1), dict(dt=F32, gdt=BF16), dict(dt=F64, gdt=F32),
                   dict(dt=BF16, gdt=F16), dict(n=-1), dict(d=-1), dict(segs=-1),
                   dict(n=2 ** 31), dict(segs=0), dict(d=2 ** 29), dict(gate=None),
                   dict(ids=None), dict(starts=None), dict(ends=None), dict(ws=P + 16)):
            assert call(**kw) == EINVAL, kw
        assert call(ws=None) == EWORKSPACE and call(nbytes=need - 1) == EWORKSPACE
    assert scan(value=None) == EINVAL and scan(dst=None) == EINVAL
    assert scan(n=0, empty=1, last=P, off=None) == EINVAL
    assert grad(g=None) == EINVAL
    assert grad(value=None) == EINVAL and grad(marks=None) == EINVAL  # for dgate
    step = lib.mdgl_segment_scan_step
    assert step(None, None, None, None, None, 0, F32, F32, None) == 0
    assert step(P, P, P, P, P, -1, F32, F32, None) == EINVAL
    assert step(P, P, P, P, P, 2 ** 40, F32, F32, None) == EINVAL
    assert step(P, P, P, P, P, 4, F32, F16, None) == EINVAL
    assert step(P, P, None, P, P, 4, F32, F32, None) == EINVAL


def test_abi_layer_norm(lib):
    ln = lib.mdgl_layer_norm
    assert ln(None, None, None, None, None, None, 0, 4, 1e-5, F32, F32, None) == 0
    assert ln(None, None, None, None, None, None, 4, 0, 1e-5, F32, F32, None) == 0
    for args in ((P, P, P, P, None, None, 4, 4, -1.0, F32, F32),
                 (P, P, P, P, None, None, 4, 4, float("nan"), F32, F32),
                 (P, P, P, P, P, None, 4, 4, 1e-5, F32, F32),
                 (P, P, P, P, None, None, -4, 4, 1e-5, F32, F32),
                 (P, P, P, P, None, None, 4, 2 ** 30, 1e-5, F32, F32),
                 (P, P, P, P, None, None, 4, 2 ** 26, 1e-5, F16, F32),
                 (P, P, P, P, None, None, 4, 4, 1e-5, F32, F64),
                 (P, P, P, P, None, None, 4, 4, 1e-5, BF16, F16),
                 (P, P, P, P, None, None, 4, 4, 1e-5, 7, 7),
                 (None, P, P, P, None, None, 4, 4, 1e-5, F32, F32),
                 (P, P, P, None, None, None, 4, 4, 1e-5, F32, F32)):
        assert ln(*args, None) == EINVAL, args
    need = lib.mdgl_layer_norm_grad_workspace_bytes(100, 40, BF16)
    assert need > 0 and lib.mdgl_layer_norm_grad_workspace_bytes(0, 40, F32) == 0
    assert lib.mdgl_layer_norm_grad_workspace_bytes(-1, 40, F32) == -1
    g = lib.mdgl_layer_norm_grad
    assert g(P, P, P, P, P, None, None, None, 100, 40, None, 0, BF16, F32, None) == 0
    assert g(P, P, P, P, P, P, P, P, 100, 40, None, 0, BF16, F32, None) == EWORKSPACE
    assert g(P, P, P, P, P, P, P, P, 100, 40, P, need - 1, BF16, F32, None) == EWORKSPACE
    assert g(P, P, P, P, P, P, P, P, 100, 40, P + 8, need, BF16, F32, None) == EINVAL
    assert g(P, P, None, P, P, P, P, P, 100, 40, P, need, BF16, F32, None) == EINVAL
    assert g(P, P, P, P, None, P, P, P, 100, 40, P, need, BF16, F32, None) == EINVAL


def test_abi_route(lib):
    def route(x=P, w=P, ids=P, n=4, e=64, k=4, score=0, groups=1, top=1, gs=0, dt=F32):
        return lib.mdgl_topk_route(x, None, w, ids, n, e, k, score, groups, top, gs, 1, 1.0, dt,
                                   None)

    assert route(n=0) == 0
    for kw in (dict(n=-1), dict(e=0), dict(e=2049), dict(k=0), dict(k=33), dict(k=65), dict(e=3),
               dict(score=2), dict(groups=0), dict(groups=7), dict(groups=65, e=130),
               dict(groups=4, top=0), dict(groups=4, top=5), dict(groups=32, top=1),
               dict(gs=2), dict(dt=4), dict(x=None), dict(w=None), dict(ids=None)):
        assert route(**kw) == EINVAL, kw
    g = lib.mdgl_topk_route_grad
    assert g(None, None, None, None, 0, 64, 4, 0, 1, 1.0, F32, None) == 0
    assert g(P, P, P, None, 4, 64, 4, 0, 1, 1.0, F32, None) == EINVAL
    assert g(P, P, P, P, 4, 64, 4, 5, 1, 1.0, F32, None) == EINVAL
    ws = lib.mdgl_route_plan_workspace_bytes
    assert ws(10, 64) == 0 and ws(1 << 20, 64) > 0
    assert ws(-1, 64) == ws(10, 0) == ws(10, 2049) == ws(2 ** 31, 4) == -1
    plan = lib.mdgl_route_plan
    assert plan(P, -1, 64, P, P, P, None, 0, None) == EINVAL
    assert plan(P, 10, 2049, P, P, P, None, 0, None) == EINVAL
    assert plan(P, 10, 64, None, P, P, None, 0, None) == EINVAL
    assert plan(None, 10, 64, P, P, P, None, 0, None) == EINVAL
    assert plan(P, 1 << 20, 64, P, P, P, None, 0, None) == EWORKSPACE
    assert plan(P, 1 << 20, 64, P, P, P, P + 4, 1 << 30, None) == EINVAL


def test_abi_moves(lib):
    d, c, g = lib.mdgl_dispatch_rows, lib.mdgl_combine_rows, lib.mdgl_combine_rows_grad
    for args in ((0, 2, 4), (4, 0, 4), (4, 2, 0)):
        assert d(None, None, None, *args, F32, None) == 0
        assert g(None, None, None, None, None, None, *args, F32, None) == 0
    assert c(None, None, None, None, 0, 2, 4, F32, None) == 0
    for args in ((-1, 2, 4), (4, -2, 4), (4, 2, -4), (2 ** 30, 2, 4), (4, 2, 2 ** 30)):
        assert d(P, P, P, *args, F32, None) == EINVAL
        assert c(P, P, P, P, *args, F32, None) == EINVAL
        assert g(P, P, P, P, P, P, *args, F32, None) == EINVAL
    assert d(P, None, P, 4, 2, 4, F32, None) == EINVAL and d(P, P, P, 4, 2, 4, 8, None) == EINVAL
    assert c(P, None, P, P, 4, 2, 4, F32, None) == EINVAL
    assert g(P, P, None, P, P, P, 4, 2, 4, F32, None) == EINVAL
    assert g(None, P, P, P, P, P, 4, 2, 4, F32, None) == EINVAL  # for dweights


def test_no_gpu_is_an_error():
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    x = np.zeros((3, 4), np.float32)
    for call in (lambda: ops.layer_norm(x), lambda: ops.segment_scan([3], x, x),
                 lambda: ops.segment_scan_step(x, x, x), lambda: ops.topk_route(x, 1),
                 lambda: ops.route_plan(np.zeros(3, np.int64), 2)):
        with pytest.raises(RuntimeError, match="no GPU"):
            call()

"""Layers of experts (the root-mean-square norm, values in 8 bits, the experts'
products) without a GPU: refusals of the Python layer before any GPU work, and of the
C ABI before a launch."""

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import mojodgl as dgl
import mojodgl.nn.functional as nnf
import mojodgl.ops as ops
from mojodgl import DGLError, _lib

F32, F64, BF16, F16, F8 = 0, 1, 2, 3, 4
EINVAL, EWORKSPACE = -1, -2
P = 4096  # an aligned address that no refused call reads


def test_names():
    assert nnf.rms_norm is ops.rms_norm is dgl.rms_norm
    for name in ("rms_norm", "Quantized", "quantize_rows", "quantize_blocks", "expert_mm",
                 "scaled_mm"):
        assert getattr(dgl, name) is getattr(ops, name) and getattr(ops, name).__doc__
        assert name in dgl.__all__ and name not in ops.__all__


def test_rms_norm_refusals():
    x = np.zeros((3, 4), np.float32)
    for bad in (np.zeros(3), np.zeros((1, 4)), np.zeros(5, np.float32)):
        with pytest.raises(DGLError, match="weight"):
            ops.rms_norm(x, bad)
    for bad in (np.zeros((3, 5)), np.zeros(4), np.zeros((1, 4))):
        with pytest.raises(DGLError, match="residual"):
            ops.rms_norm(x, None, bad)
    with pytest.raises(DGLError, match="axes"):
        ops.rms_norm(np.float32(1.0))
    with pytest.raises(DGLError, match="complex"):
        ops.rms_norm(x.astype(np.complex64))
    for eps in (-1.0, float("nan")):
        with pytest.raises(DGLError, match="eps"):
            ops.rms_norm(x, eps=eps)
    for args in ((x.astype(np.float64),), (x, x[0].astype(np.float64)),
                 (x, None, x.astype(np.float64))):
        with pytest.raises(DGLError, match="float64"):
            ops.rms_norm(*args, quantize=True)
    with pytest.raises(DGLError, match="no gradient"):
        ops.rms_norm(torch.zeros(3, 4), torch.ones(4, requires_grad=True), quantize=True)


def test_quantize_refusals():
    x = np.zeros((3, 4), np.float32)
    for call in (ops.quantize_rows, ops.quantize_blocks):
        with pytest.raises(DGLError, match="float64"):
            call(x.astype(np.float64))
        with pytest.raises(DGLError, match="no gradient"):
            call(torch.zeros(3, 4, requires_grad=True))
        with pytest.raises(DGLError, match="complex"):
            call(x.astype(np.complex64))
        with pytest.raises(DGLError, match="quantized"):
            call(ops.Quantized(torch.zeros(3, 4), torch.zeros(3, 1)))
    with pytest.raises(DGLError, match="axes"):
        ops.quantize_rows(np.float32(1))
    with pytest.raises(DGLError, match="matrices"):
        ops.quantize_blocks(x[0])


def quantized(*shape, axes=1):
    scale = shape[:-axes] + tuple(-(-d // 128) for d in shape[-axes:])
    return ops.Quantized(torch.zeros(shape).to(torch.float8_e4m3fn), torch.ones(scale))


def test_expert_mm_refusals():
    x, w = np.zeros((5, 4), np.float32), np.zeros((2, 4, 3), np.float32)
    for a, b in ((x[0], w), (x, w[0]), (x[None], w)):
        with pytest.raises(DGLError, match="shape"):
            ops.expert_mm(a, b, [2, 3])
    with pytest.raises(DGLError, match="inner dimensions"):
        ops.expert_mm(x[:, :3], w, [2, 3])
    with pytest.raises(DGLError, match="one type"):
        ops.expert_mm(x, w.astype(np.float64), [2, 3])
    with pytest.raises(DGLError, match="one type"):
        ops.expert_mm(torch.zeros(5, 4, dtype=torch.bfloat16), torch.zeros(2, 4, 3), [2, 3])
    for lens in ([2], [1, 2, 2], [[2, 3]]):
        with pytest.raises(DGLError, match="one length for each"):
            ops.expert_mm(x, w, lens)
    for lens in ([-1, 3], [3, 3], [2 ** 62, 2 ** 62], [6, -1]):
        with pytest.raises(DGLError, match="lengths must be"):
            ops.expert_mm(x, w, lens)
    with pytest.raises(DGLError, match="whole numbers"):
        ops.expert_mm(x, w, [0.5, 1.0])


def test_scaled_mm_refusals():
    x, w = quantized(5, 200), quantized(2, 200, 3, axes=2)
    with pytest.raises(DGLError, match="quantize_blocks"):
        ops.scaled_mm(x, torch.zeros(2, 200, 3), [2, 3])
    for bad in (ops.Quantized(x.data, x.scale[:, :1]), ops.Quantized(x.data, x.scale[:4]),
                ops.Quantized(x.data, x.scale.double()), ops.Quantized(x.data.float(), x.scale),
                ops.Quantized(x.data, None)):
        with pytest.raises(DGLError, match="scale"):
            ops.scaled_mm(bad, w, [2, 3])
    for bad in (ops.Quantized(w.data, w.scale[:, :1]), ops.Quantized(w.data, w.scale[..., 0]),
                ops.Quantized(w.data.float(), w.scale)):
        with pytest.raises(DGLError, match="scale"):
            ops.scaled_mm(x, bad, [2, 3])
    with pytest.raises(DGLError, match="inner dimensions"):
        ops.scaled_mm(quantized(5, 199), w, [2, 3])
    with pytest.raises(DGLError, match="plan or lengths"):
        ops.scaled_mm(x, w)
    with pytest.raises(DGLError, match="one length for each"):
        ops.scaled_mm(x, w, [5])
    with pytest.raises(DGLError, match="lengths must be"):
        ops.scaled_mm(x, w, [5, 1])
    with pytest.raises(DGLError, match="dtype"):
        ops.scaled_mm(x, w, [2, 3], dtype=torch.float64)
    with pytest.raises(DGLError, match="float64"):
        ops.scaled_mm(np.zeros((5, 200)), w, [2, 3])
    with pytest.raises(DGLError, match="shape"):
        ops.scaled_mm(quantized(1, 5, 200), w, [2, 3])
    with pytest.raises(DGLError, match="shape"):
        ops.scaled_mm(x, quantized(1, 2, 200, 3, axes=2), [2, 3])


def test_tangents_are_refused():
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.ones(4, 3), torch.ones(4, 3))
        y = torch.ones(4, 3)
        for call in (lambda: ops.rms_norm(x), lambda: ops.rms_norm(y, x[0]),
                     lambda: ops.rms_norm(y, None, x), lambda: ops.rms_norm(x, quantize=True),
                     lambda: ops.quantize_rows(x), lambda: ops.quantize_blocks(x),
                     lambda: ops.expert_mm(x, torch.ones(1, 3, 2), [4]),
                     lambda: ops.scaled_mm(x, quantized(3, 2, axes=2))):
            with pytest.raises(DGLError, match="tangent"):
                call()


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def test_abi_rms_norm(lib):
    def norm(x=P, r=P, w=P, y=P, scale=None, total=P, rstd=None, n=4, d=4, eps=1e-6, dt=F32,
             wdt=F32, rdt=F32):
        return lib.mdgl_rms_norm(x, r, w, y, scale, total, rstd, n, d, eps, dt, wdt, rdt, None)

    assert norm(n=0) == norm(d=0) == 0
    for kw in (dict(eps=-1.0), dict(eps=float("nan")), dict(n=-1), dict(d=-1), dict(d=2 ** 26),
               dict(dt=F8), dict(dt=-1), dict(wdt=F64), dict(rdt=BF16), dict(rdt=F64),
               dict(dt=BF16, wdt=F16), dict(dt=BF16, rdt=F16), dict(dt=F64), dict(x=None),
               dict(y=None), dict(total=None),
               dict(dt=F64, wdt=F64, rdt=F64, scale=P)):
        assert norm(**kw) == EINVAL, kw
    ws = lib.mdgl_rms_norm_grad_workspace_bytes
    need = ws(100, 40, BF16)
    assert need > 0 and ws(0, 40, F32) == ws(4, 0, F32) == 0
    assert ws(-1, 40, F32) == ws(4, -1, F32) == ws(4, 4, F8) == -1

    def grad(t=P, r=None, rstd=P, g=P, dx=P, dr=None, dw=P, n=100, d=40, w=P, nbytes=need,
             dt=BF16, wdt=F32, rdt=BF16):
        return lib.mdgl_rms_norm_grad(t, r, P, rstd, g, None, dx, dr, dw, n, d, w, nbytes, dt,
                                      wdt, rdt, None)

    assert grad(n=0) == grad(d=0) == grad(dx=None, dw=None) == 0
    assert grad(w=None) == grad(nbytes=need - 1) == EWORKSPACE
    for kw in (dict(t=None), dict(rstd=None), dict(g=None), dict(w=P + 8), dict(n=-1),
               dict(rdt=F32, r=P), dict(dt=F32, rdt=F32, r=P), dict(rdt=F16), dict(dt=7)):
        assert grad(**kw) == EINVAL, kw


def test_abi_quantize(lib):
    rows, mats = lib.mdgl_quantize_rows, lib.mdgl_quantize_blocks
    assert rows(None, None, None, 0, 4, F32, None) == rows(None, None, None, 4, 0, F32, None) == 0
    for args in ((P, P, P, 4, 4, F64), (P, P, P, 4, 4, F8), (P, P, P, -1, 4, F32),
                 (P, P, P, 4, -1, F32), (None, P, P, 4, 4, F32), (P, None, P, 4, 4, F32),
                 (P, P, None, 4, 4, F32), (P, P, P, 4, 2 ** 29, F32)):
        assert rows(*args, None) == EINVAL, args
    for sizes in ((0, 4, 4), (4, 0, 4), (4, 4, 0)):
        assert mats(None, None, None, *sizes, 0, F32, None) == 0
    for args in ((P, P, P, 1, 4, 4, 0, F64), (P, P, P, -1, 4, 4, 0, F32),
                 (P, P, P, 1, -4, 4, 0, F32), (P, P, P, 1, 4, -4, 1, F32),
                 (P, P, P, 1, 2 ** 20, 2 ** 20, 0, F32), (None, P, P, 1, 4, 4, 0, F32),
                 (P, None, P, 1, 4, 4, 0, F32), (P, P, None, 1, 4, 4, 0, F32)):
        assert mats(*args, None) == EINVAL, args


def test_abi_expert_mm(lib):
    ws = lib.mdgl_expert_mm_workspace_bytes
    assert ws(0, 4, 2, 4, BF16) == ws(5, 4, 2, 0, F16) == 0
    for args in ((-1, 4, 2, 4, BF16), (5, -1, 2, 4, BF16), (5, 4, -1, 4, BF16), (5, 4, 2, -1, BF16),
                 (5, 4, 2, 4, F32), (5, 4, 2, 4, F8), (2 ** 31, 4, 2, 4, BF16),
                 (5, 2 ** 20, 2, 4, BF16), (5, 4, 2, 2 ** 20, BF16), (5, 4, 65536, 4, BF16),
                 (2 ** 31 - 1, 4, 2, 2 ** 20 - 1, BF16)):
        assert ws(*args) == -1, args

    def mm(a=P, b=P, y=P, lens=P, n=5, d1=8, r=2, d2=8, t=0, w=P, nbytes=1 << 40, dt=BF16):
        return lib.mdgl_expert_mm(a, b, y, lens, n, d1, r, d2, t, w, nbytes, dt, None)

    assert mm(n=0) == mm(d2=0) == 0
    for kw in (dict(dt=F32), dict(dt=F64), dict(dt=F8), dict(n=-1), dict(d1=-1), dict(r=-1),
               dict(d2=-1), dict(n=2 ** 31), dict(d1=2 ** 20), dict(d2=2 ** 20), dict(r=65536),
               dict(a=None), dict(b=None), dict(y=None), dict(lens=None),
               dict(n=2 ** 31 - 1, d2=2 ** 20 - 8)):
        assert mm(**kw) == EINVAL, kw

    gws = lib.mdgl_expert_mm_grad_workspace_bytes
    assert gws(5, 4, 0, 4, BF16) == gws(5, 0, 2, 4, BF16) == 0
    need = gws(100000, 8, 1, 8, BF16)
    assert need > 0 and gws(5, 4, 2, 4, F32) == gws(-1, 4, 2, 4, BF16) == -1
    assert gws(5, 2 ** 20 - 1, 65535, 2 ** 20 - 1, BF16) == -1

    def grad(a=P, g=P, db=P, lens=P, n=100000, d1=8, r=1, d2=8, w=P, nbytes=need, dt=BF16):
        return lib.mdgl_expert_mm_grad(a, g, db, lens, n, d1, r, d2, w, nbytes, dt, None)

    assert grad(r=0) == grad(d1=0) == grad(d2=0) == 0
    assert grad(w=None) == grad(nbytes=need - 1) == EWORKSPACE
    for kw in (dict(dt=F32), dict(n=-1), dict(r=65536), dict(a=None), dict(g=None), dict(db=None),
               dict(lens=None), dict(w=P + 16)):
        assert grad(**kw) == EINVAL, kw


def test_abi_scaled_mm(lib):
    ws = lib.mdgl_scaled_mm_workspace_bytes
    assert ws(0, 4, 2, 4) == 0 and ws(-1, 4, 2, 4) == ws(5, 4, 65536, 4) == -1

    def mm(a=P, sa=P, b=P, sb=P, y=P, lens=P, n=5, d1=16, r=2, d2=8, w=P, nbytes=1 << 40, dt=BF16):
        return lib.mdgl_scaled_mm(a, sa, b, sb, y, lens, n, d1, r, d2, w, nbytes, dt, None)

    assert mm(n=0) == mm(d2=0) == 0
    for kw in (dict(dt=F64), dict(dt=F8), dict(n=-1), dict(d1=2 ** 20), dict(r=65536),
               dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(y=None),
               dict(lens=None), dict(lens=None, r=0)):
        assert mm(**kw) == EINVAL, kw
    # bytes can be dispatched, not combined
    d, c = lib.mdgl_dispatch_rows, lib.mdgl_combine_rows
    assert d(None, None, None, 0, 2, 4, F8, None) == 0
    assert d(P, None, P, 4, 2, 4, F8, None) == EINVAL
    assert c(P, P, P, P, 4, 2, 4, F8, None) == EINVAL


def test_no_gpu_is_an_error():
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible")
    x = np.zeros((3, 4), np.float32)
    for call in (lambda: ops.rms_norm(x), lambda: ops.quantize_rows(x),
                 lambda: ops.quantize_blocks(x), lambda: ops.expert_mm(x, x[None, :, :3].repeat(
                     2, 0).reshape(1, 6, 3)[:, :4], [3]),
                 lambda: ops.scaled_mm(x, quantized(4, 2, axes=2))):
        with pytest.raises(RuntimeError, match="no GPU"):
            call()

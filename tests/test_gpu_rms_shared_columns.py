"""Columns that two lanes of the root-mean-square norm hold (rows whose width is no
multiple of a vector): what is no number in one of them touches the results that the
definition says, and no others. An infinite value makes its row's 1 / rms 0, so the row's
other results are 0, its own NaN, and the weight's gradient NaN in its column alone."""

import pytest
import torch

import mojodgl.ops as ops

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
HALF_STEP = {F32: 2.0 ** -24, F64: 2.0 ** -53, BF16: 2.0 ** -8, F16: 2.0 ** -11}
INF = float("inf")
VECTOR = {F32: 4, F64: 2, BF16: 8, F16: 8}
# a width of each way that rows lie on threads
WIDTHS = [17, 43, 61, 125, 253, 301, 603, 1021, 1501, 3001, 7999, 16381]
ROW = 2


def shared(d, dtype):
    """Columns in the last two vectors of a row."""
    return range(d - VECTOR[dtype], d // VECTOR[dtype] * VECTOR[dtype])


def rows(d, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g, device="cuda", dtype=F64).to(dtype)  # noqa: E731
    return make(5, d), make(d), make(5, d), make(5, d)


@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("d", WIDTHS)
def test_infinity_in_a_shared_column(dtype, d):
    assert len(shared(d, dtype)) > 0
    x, w, r, dy = rows(d, dtype, d)
    for at in {shared(d, dtype)[0], shared(d, dtype)[-1]}:
        for value in (INF, -INF):
            x[ROW, at] = value
            others = torch.arange(d, device="cuda") != at
            X, W, R = (t.clone().requires_grad_() for t in (x, w, r))
            y, total = ops.rms_norm(X, W, R)
            assert y[ROW, at].isnan() and (y[ROW, others] == 0).all()
            assert total[ROW, at] == value and total[ROW, others].isfinite().all()
            finite = torch.arange(5, device="cuda") != ROW
            assert y[finite].isfinite().all()
            dx, dw, dr = torch.autograd.grad(y, (X, W, R), dy)
            assert dw[at].isnan()
            # the finite rows' terms alone: the row's own are 0
            t = x[finite].double() + r[finite].double()
            xh = t / (t.square().mean(1, keepdim=True) + 1e-6).sqrt()
            want = (dy[finite].double() * xh).sum(0)[others]
            size = (dy[finite].double() * xh).abs().sum(0)[others]
            # the root's sum passes at most 48 + d / 1024 roundings and 12 around it, dw
            # at most 160 (test_gpu_rms_quant: relative, bounds); then its own
            u = HALF_STEP[F64 if dtype == F64 else F32]
            bound = (60 + d / 1024 + 160) * u * size
            h = HALF_STEP[dtype]
            assert ((dw[others].double() - want).abs()
                    <= bound * (1 + h) + want.abs() * h + 2.0 ** -24 * (dtype == F16)).all()
            assert dx[finite].isfinite().all() and dr[finite].isfinite().all()
            if dtype == F64:
                continue
            q, _ = ops.rms_norm(x, w, r, quantize=True)
            data = q.data.float()
            assert data[ROW, at].isnan() and (data[ROW, others] == 0).all()
            assert (q.scale[ROW] == 2.0 ** -126).all()
            assert data[finite].isfinite().all() and q.scale.isfinite().all()
        x[ROW, at] = 1.0


@pytest.mark.parametrize("dtype", [F32, F64, BF16])
@pytest.mark.parametrize("d", WIDTHS)
def test_infinite_normalised_values(dtype, d):
    """A row whose squares all lie below the range, with eps = 0: 1 / rms is infinite, so
    are its normalised values, and by the definition (gradients and weights above 0) its
    gradient is inf * (g - inf * inf) = -inf in every column. (float16 has no such values.)"""
    x, w, _, _ = rows(d, dtype, d)
    x[ROW] = 2.0 ** (-600 if dtype == F64 else -100)
    X, W = x.requires_grad_(), (w.abs() + 1.0).requires_grad_()
    y = ops.rms_norm(X, W, eps=0.0)
    assert (y[ROW] == INF).all()
    dx, dw = torch.autograd.grad(y, (X, W), torch.ones_like(y))
    assert (dw == INF).all()  # one infinite term in each column's sum
    assert (dx[ROW] == -INF).all()
    finite = torch.arange(5, device="cuda") != ROW
    assert dx[finite].isfinite().all()

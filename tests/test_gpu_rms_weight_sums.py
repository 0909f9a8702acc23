"""How near the gradient of rms_norm's weight, a sum over all rows in float32, comes to
float64 for many rows.

An addition in float32 that gives S is off by a value spread over half a step of S at most,
u |S| with u = 2^-24: in the mean square by u^2 S^2 / 3. In a chain of L independent terms of
variance v S^2 is i v behind the i-th, so the chain is off by u^2 L^2 v / 6 in the mean square,
a share of L u^2 / 6 of its own L v. dw passes chains of 16 rows, their L / 16 sums, up to 64
workgroups' sums and 16 of those (a column's 16 threads), besides the rounding of xh and of
1 / rms (less than 2 u^2 together): the root mean square of dw's error over its columns is at
most sqrt((16 + L / 16 + 64 + 16) / 6 + 2) u of that of dw. One chain of L = 200 rows in
place of the first two comes to 5 u and more."""

import pytest
import torch

import mojodgl.ops as ops

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("dtype,d,rows,workgroups", [
    (F32, 520, 1, 1024), (F32, 1500, 1, 1024), (F32, 3000, 1, 512), (F32, 8200, 1, 512),
    (F32, 16000, 1, 256), (F32, 40, 16, 1024), (F32, 400, 4, 1024), (BF16, 1040, 1, 1024),
    (BF16, 4096, 1, 1024), (BF16, 8000, 1, 512), (BF16, 16384, 1, 512)])
@pytest.mark.parametrize("residual", [False, True])
def test_sums_of_many_rows(dtype, d, rows, workgroups, residual):
    """`workgroups` of a card's worth take `rows` rows at a time."""
    if rows > 1 and residual:
        pytest.skip("the same sums")
    length = 200
    n = length * rows * workgroups + 3
    g = torch.Generator(device="cuda").manual_seed(d)
    x, dy = (torch.randn(n, d, generator=g, device="cuda", dtype=dtype) for _ in range(2))
    r = torch.randn(n, d, generator=g, device="cuda", dtype=dtype) if residual else None
    w = torch.ones(d, device="cuda", requires_grad=True)
    y = ops.rms_norm(x, w, r)
    dw, = torch.autograd.grad(y[0] if residual else y, w, dy)
    want = torch.zeros(d, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 27) // d)
    for i in range(0, n, step):
        t = x[i:i + step].double()
        if residual:
            t += r[i:i + step]
        t /= (t.square().mean(1, keepdim=True) + 1e-6).sqrt()
        want += (t * dy[i:i + step]).sum(0)
    off = ((dw.double() - want).square().mean() / want.square().mean()).sqrt().item()
    assert off <= ((16 + length / 16 + 64 + 16) / 6 + 2) ** 0.5 * 2.0 ** -24, off * 2 ** 24


def test_rows_wider_than_registers():
    """One thread a column, 64 runs of rows: chains of 16 rows, their sums, 4 and 16 of the
    runs'."""
    n, d = 64 * 312, 16400
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(n, d, generator=g, device="cuda") for _ in range(2))
    w = torch.ones(d, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(ops.rms_norm(x, w), w, dy)
    want = torch.zeros(d, dtype=torch.float64, device="cuda")
    for i in range(0, n, 2048):
        t = x[i:i + 2048].double()
        t /= (t.square().mean(1, keepdim=True) + 1e-6).sqrt()
        want += (t * dy[i:i + 2048]).sum(0)
    off = ((dw.double() - want).square().mean() / want.square().mean()).sqrt().item()
    assert off <= ((16 + 312 / 16 + 4 + 16) / 6 + 2) ** 0.5 * 2.0 ** -24, off * 2 ** 24

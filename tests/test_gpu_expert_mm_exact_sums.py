"""Sums of whole numbers, which float32 holds exactly: the experts' products and their
gradients are the exact sums rounded once, to the last bit, where the inner axis goes in
parts and a group's rows in pieces, too. A part or a piece that passed through fewer bits, or
a term left out or counted twice, would show."""

import pytest
import torch

import mojodgl.ops as ops

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
F8 = torch.float8_e4m3fn

#: lengths, rows behind, d1, d2: few rows of a long inner axis (in 8, 4 and 2 parts), widths
#: that end inside a piece of 16 bytes, tiles of each size, long groups of few tiles
SHAPES = [([64], 0, 4096, 4096), ([20, 0, 11], 3, 4099, 48), ([1], 0, 8191, 16),
          ([100, 28], 0, 1030, 136), ([700, 20, 900], 10, 264, 328), ([8192], 0, 64, 64),
          ([5000, 0, 3000], 5, 300, 202), ([9000, 77], 0, 301, 203), ([3000, 5200], 0, 72, 4104),
          ([2500, 2500], 0, 1030, 2050)]


def whole(g, low, high, *shape):
    return torch.randint(low, high + 1, shape, generator=g, device="cuda").double()


def products(x, w, lens):
    y, at = x.new_zeros(x.shape[0], w.shape[2]), 0
    for e, m in enumerate(lens):
        y[at:at + m] = x[at:at + m] @ w[e]
        at += m
    return y


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_products_and_gradients(shape, turned, dtype):
    """Terms of at most 8 * 6: sums of up to 9,000 of them stay below 2^24, and, of mean 0,
    within float16's range."""
    lens, behind, d1, d2 = SHAPES[shape]
    g = torch.Generator(device="cuda").manual_seed(shape)
    n, r = sum(lens) + behind, len(lens)
    x, w, dy = whole(g, -8, 8, n, d1), whole(g, -6, 6, r, d1, d2), whole(g, -6, 6, n, d2)
    X = x.to(dtype).requires_grad_()
    W = w.to(dtype)
    if turned:
        W = W.transpose(1, 2).contiguous().transpose(1, 2)
    W.requires_grad_()
    y = ops.expert_mm(X, W, lens)
    want = products(x, w, lens)
    assert want.abs().max() > 256  # more bits than bfloat16 has
    assert torch.equal(y.detach(), want.to(dtype))
    dx, dw = torch.autograd.grad(y, (X, W), dy.to(dtype))
    assert torch.equal(dx, products(dy, w.transpose(1, 2).contiguous(), lens).to(dtype))
    want, at = torch.zeros_like(w), 0
    for e, m in enumerate(lens):
        want[e] = x[at:at + m].t().contiguous() @ dy[at:at + m]
        at += m
    assert torch.equal(dw, want.to(dtype))


@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_products_in_8_bits(shape):
    """Values of 0, 1 and 2 in size: products of 2^0 to 2^2, which the matrix cores add
    whole; scales are powers of two."""
    lens, behind, d1, d2 = SHAPES[shape]
    g = torch.Generator(device="cuda").manual_seed(shape)
    n, r = sum(lens) + behind, len(lens)
    x, w = whole(g, -2, 2, n, d1), whole(g, -2, 2, r, d1, d2)
    b1, b2 = -(-d1 // 128), -(-d2 // 128)
    sx, sw = 2.0 ** whole(g, -2, 1, n, b1), 2.0 ** whole(g, -1, 2, r, b1, b2)
    spread = lambda s, d, axis: s.repeat_interleave(128, axis).narrow(axis, 0, d)  # noqa: E731
    want = products(x * spread(sx, d1, 1), w * spread(spread(sw, d1, 1), d2, 2), lens)
    q = ops.Quantized(x.to(F8), sx.float())
    v = ops.Quantized(w.transpose(1, 2).contiguous().to(F8).transpose(1, 2), sw.float())
    assert torch.equal(ops.scaled_mm(q, v, lens, dtype=F32).double(), want)
    assert torch.equal(ops.scaled_mm(q, v, lens, dtype=BF16), want.to(BF16))

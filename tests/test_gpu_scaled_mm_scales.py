"""scaled_mm at the ends of its scales' range: two scales that float32 holds while their
product is past its range or below it, scales of 0, subnormal and negative ones, against
float64 and with the tolerances of test_gpu_expert_mm."""

import pytest
import torch

import mojodgl.ops as ops
from test_gpu_expert_mm import F8, F16, F32, BF16, U, check, cut, gen, products, rand, values

pytestmark = pytest.mark.gpu

#: lengths, d1, d2: tiles of each size, widths that end inside a piece of 16 bytes, and few
#: rows of a long inner axis, which goes in parts
SHAPES = [([5], 256, 40), ([40, 0, 25], 250, 130), ([300, 170], 640, 257), ([64], 4096, 512),
          ([31], 2065, 48), ([3000, 2500], 512, 1100), ([3000, 2500], 509, 1030)]


def quantized(g, kind, n, r, d1, d2):
    """Rows and matrices of that kind of scales; b is a block of the inner axis."""
    b, c = -(-d1 // 128), -(-d2 // 128)
    one = lambda *s: 1.0 + torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    sx, sw = one(n, b), one(r, b, c)
    x, w = rand(g, n, d1), rand(g, r, d1, d2)
    if kind in ("above", "some above"):
        # products of the scales of 2^128 to 2^130; a block's sum is at most 128 * 2^-16
        x, w = x.clamp(-1, 1) * 2.0 ** -8, w.clamp(-1, 1) * 2.0 ** -8
        x[::2, :128] = 0.0  # whose sums are 0 in the first block
        sx, sw = sx * 2.0 ** 64, sw * 2.0 ** 64
        if kind == "some above":  # in one block of some rows, far from the others' sizes
            sx[:, :] = one(n, b) * 2.0 ** -60
            sx[::7, b // 2] = 2.0 ** 64.5
    elif kind == "below":
        # products of 2^-149 to 2^-147, sums of a block of about 2^23
        x, w = 256 * (1 + x.abs().clamp_max(0.75)), 256 * (1 + w.abs().clamp_max(0.75))
        sx, sw = sx * 2.0 ** -75, sw * 2.0 ** -74
    else:
        # one far above 1, the other far below; 0, subnormal and negative ones among them
        k = torch.randint(-120, 121, (b,), generator=g, device="cuda").float()
        sx, sw = sx * 2.0 ** k, sw * (2.0 ** -k).unsqueeze(1)
        sx[::3, 0], sw[:, 0] = 0.0, sw[:, 0] / sw[:, 0] * 1.5 * 2.0 ** 127
        sx[1::3, 0] = 3 * 2.0 ** -146
        sx[2::3, 0] = -(2.0 ** -126)
    w = w.to(F8).transpose(1, 2).contiguous().transpose(1, 2)
    return ops.Quantized(x.to(F8), sx), ops.Quantized(w, sw)


def allowed(qx, qw, lens, size):
    """test_gpu_expert_mm's bound. What is cut off is a share of the terms' sizes: it takes
    the scales without their signs (with them it would be below 0). Besides, a product of
    scales below 2^-126 is rounded to a multiple of 2^-149: for each block half of that
    times its sum, 128 * 448^2 at most."""
    bare = [ops.Quantized(q.data, q.scale.abs()) for q in (qx, qw)]
    return (qx.data.shape[1] + 64 + 4) * U * size + cut(*bare, lens) \
        + qx.scale.shape[1] * 2.0 ** -150 * 128 * 448 ** 2


@pytest.mark.parametrize("kind", ["above", "some above", "below", "apart"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_products_of_scales_out_of_range(shape, kind):
    lens, d1, d2 = SHAPES[shape]
    g = gen(shape)
    qx, qw = quantized(g, kind, sum(lens), len(lens), d1, d2)
    assert qx.scale.isfinite().all() and qw.scale.isfinite().all()
    want, size = products(values(qx, (1,)), values(qw, (1, 2)), lens)
    assert (want.abs() < 2.0 ** 127).all()
    y = ops.scaled_mm(qx, qw, lens, dtype=F32)
    assert y.isfinite().all()
    bound = allowed(qx, qw, lens, size)
    check(y, want, bound, kind)
    if kind == "above":  # bfloat16 has float32's range, float16 has not
        check(ops.scaled_mm(qx, qw, lens, dtype=BF16), want, bound, kind)
        half = ops.scaled_mm(qx, qw, lens, dtype=F16)
        assert (half[want.abs() > 2.0 ** 17].isinf()).all() and not half.isnan().any()


@pytest.mark.parametrize("d1", [256, 250])
def test_infinite_scales(d1):
    """Beside rows whose scales' products leave the range: a row with an infinite scale is
    infinite or NaN (0 times it), and others are as they are without it."""
    g = gen(d1)
    qx, qw = quantized(g, "above", 300, 1, d1, 200)
    clean = ops.scaled_mm(qx, qw, [300], dtype=F32)
    qx.scale[7, 1], qx.scale[280, 0] = float("inf"), float("nan")
    y = ops.scaled_mm(qx, qw, [300], dtype=F32)
    fine = torch.ones(300, dtype=torch.bool, device="cuda")
    fine[7] = fine[280] = False
    assert clean.isfinite().all() and torch.equal(y[fine], clean[fine])
    assert not y[7].isfinite().any() and y[280].isnan().all()


def test_results_past_the_range_are_infinite():
    """Scales whose results are, by the definition, past float32's range."""
    x = torch.ones(3, 128, device="cuda").to(F8)
    w = torch.ones(1, 16, 128, device="cuda").to(F8).transpose(1, 2)
    x[1] = (-x[1].float()).to(F8)
    big = torch.full((3, 1), 2.0 ** 100, device="cuda")
    y = ops.scaled_mm(ops.Quantized(x, big), ops.Quantized(w, big[:1].reshape(1, 1, 1)), [3],
                      dtype=F32)
    inf = float("inf")
    assert (y[0] == inf).all() and (y[1] == -inf).all() and (y[2] == inf).all()

"""The experts' products in 16 bits (and the wider types), their gradients, and the
products in 8 bits, on the GPU against plain float64.

u is half a step of float32 (2^-24). Products of two 16-bit or two e4m3 values are exact
in float32; a sum of K of them is off by at most (K + 64) u times the sum of their sizes
(and in 8 bits by what `cut` says), and is rounded to the result's type once (half a step
of it)."""

import pytest
import torch

import mojodgl.ops as ops
from mojodgl import DGLError

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
F8 = torch.float8_e4m3fn
HALF_STEP = {F32: 2.0 ** -24, F64: 2.0 ** -53, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -126, F64: 0.0, BF16: 2.0 ** -126, F16: 2.0 ** -24}
U = 2.0 ** -24
NAN, INF = float("nan"), float("inf")


def check(got, want, bound, name):
    assert got.shape == want.shape, name
    h = HALF_STEP[got.dtype]
    limit = bound * (1 + h) + want.abs() * h + TINY[got.dtype]
    off = (got.double() - want).abs()
    worst = int((off - limit).argmax()) if off.numel() else 0
    assert bool((off <= limit).all()), "{}: off by {} where {} is allowed, at {} of {}".format(
        name, off.reshape(-1)[worst].item(), limit.reshape(-1)[worst].item(), worst,
        tuple(got.shape))


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=F64).to(dtype)


def groups_of(lens):
    at = 0
    for e, m in enumerate(lens):
        yield e, slice(at, at + m)
        at += m


def products(x, w, lens):
    """(products, sums of the terms' sizes) in float64."""
    x, w = x.double(), w.double()
    y, size = (x.new_zeros(x.shape[0], w.shape[2]) for _ in range(2))
    for e, at in groups_of(lens):
        y[at] = x[at] @ w[e]
        size[at] = x[at].abs() @ w[e].abs()
    return y, size


def weight_gradients(x, g, lens, r):
    x, g = x.double(), g.double()
    dw, size = (x.new_zeros(r, x.shape[1], g.shape[1]) for _ in range(2))
    for e, at in groups_of(lens):
        dw[e] = x[at].t().contiguous() @ g[at]
        size[e] = x[at].abs().t().contiguous() @ g[at].abs()
    return dw, size


# lengths (rows behind them: the last number), d1, d2
SHAPES = [
    ([1], 0, 1, 1), ([1], 0, 8, 8), ([3], 0, 64, 128), ([0, 5, 0], 2, 7, 5), ([0, 0], 4, 16, 16),
    ([17, 0, 130, 1], 9, 72, 136), ([17, 0, 130, 1], 9, 71, 135), ([64, 64, 64], 0, 64, 64),
    ([128, 128], 0, 128, 128), ([127, 129, 1], 63, 136, 120), ([300], 0, 1000, 40),
    ([33, 65, 200], 0, 602, 301), ([33, 65, 200], 5, 602, 300), ([50, 0, 70], 0, 24, 1030),
    ([0] * 63 + [5, 7] + [0] * 70 + [9], 3, 40, 48), (list(range(70)), 0, 33, 24),
    ([2] * 200, 1, 136, 264), ([700, 20, 900], 10, 264, 328), ([4096], 0, 64, 64),
    ([5000, 30], 0, 130, 66), ([1, 0, 2, 1], 0, 2048, 1408), ([8192], 0, 128, 4096),
    ([3000, 0, 5200], 100, 72, 4104), ([2500, 2500], 0, 1030, 2050),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32, F64])
@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_expert_mm(shape, turned, dtype):
    lens, behind, d1, d2 = SHAPES[shape]
    g = gen(shape)
    n, r = sum(lens) + behind, len(lens)
    u = HALF_STEP[F64] if dtype == F64 else U
    # float32 products leave out parts of 2^-24 of a term at most: one rounding more
    extra = 64 if dtype != F32 else 65
    x, dy = rand(g, n, d1, dtype=dtype), rand(g, n, d2, dtype=dtype)
    w = rand(g, r, d1, d2, dtype=dtype)
    if turned:
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    X, W = x.clone().requires_grad_(), w.detach().requires_grad_()
    y = ops.expert_mm(X, W, lens)
    assert y.dtype == dtype and torch.equal(ops.expert_mm(x, w, lens), y.detach())
    want, size = products(x, w, lens)
    check(y.detach(), want, (d1 + extra) * u * size, "y")
    assert not y[sum(lens):].any()
    dx, dw = torch.autograd.grad(y, (X, W), dy)
    want, size = products(dy, w.transpose(1, 2).contiguous(), lens)
    check(dx, want, (d2 + extra) * u * size, "dx")
    assert not dx[sum(lens):].any()
    want, size = weight_gradients(x, dy, lens, r)
    most = max(lens)
    check(dw, want, (most + extra) * u * size, "dw")
    # by a plan, whose lengths the host does not see
    ids = torch.repeat_interleave(torch.arange(r + 1), torch.tensor(lens + [behind])).cuda()
    plan = ops.route_plan(ids, r)
    assert torch.equal(ops.expert_mm(x, w, plan), y.detach())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_tiles_of_every_product(dtype):
    """Sizes that the tiles of 256 by 256 take, with odd ends of rows and columns."""
    g = gen(1)
    lens, d1, d2 = [9001, 0, 7900, 3], 2056, 1544
    n = sum(lens) + 77
    x, dy = rand(g, n, d1, dtype=dtype), rand(g, n, d2, dtype=dtype)
    w = rand(g, 4, d1, d2, dtype=dtype)
    X, W = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = ops.expert_mm(X, W, lens)
    dx, dw = torch.autograd.grad(y, (X, W), dy)
    want, size = products(x, w, lens)
    check(y.detach(), want, (d1 + 64) * U * size, "y")
    want, size = products(dy, w.transpose(1, 2).contiguous(), lens)
    check(dx, want, (d2 + 64) * U * size, "dx")
    want, size = weight_gradients(x, dy, lens, 4)
    check(dw, want, (max(lens) + 64) * U * size, "dw")
    again = torch.autograd.grad(ops.expert_mm(X, W, lens), (X, W), dy)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_large_tiles_of_odd_widths(dtype):
    g = gen(11)
    lens, d1, d2 = [9001, 0, 700, 3], 2049, 2051
    n = sum(lens) + 5
    x, dy = rand(g, n, d1, dtype=dtype), rand(g, n, d2, dtype=dtype)
    w = rand(g, 4, d1, d2, dtype=dtype)
    X, W = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = ops.expert_mm(X, W, lens)
    dx, dw = torch.autograd.grad(y, (X, W), dy)
    want, size = products(x, w, lens)
    check(y.detach(), want, (d1 + 64) * U * size, "y")
    want, size = products(dy, w.transpose(1, 2).contiguous(), lens)
    check(dx, want, (d2 + 64) * U * size, "dx")
    want, size = weight_gradients(x, dy, lens, 4)
    check(dw, want, (max(lens) + 64) * U * size, "dw")
    qx, qw = ops.quantize_rows(x), ops.quantize_blocks(w)
    y = ops.scaled_mm(qx, qw, lens, dtype=F32)
    want, size = products(values(qx, (1,)), values(qw, (1, 2)), lens)
    check(y, want, (d1 + 68) * U * size + cut(qx, qw, lens), "8 bits")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d1,d2", [(72, 40), (71, 41), (136, 264)])
def test_what_is_not_a_number_stays_in_its_row(dtype, d1, d2):
    """NaN and infinities in one group's rows, at its borders, and behind the last."""
    g = gen(2)
    lens, behind = [70, 0, 130, 60], 20
    n = sum(lens) + behind
    x, dy = rand(g, n, d1, dtype=dtype), rand(g, n, d2, dtype=dtype)
    w = rand(g, 4, d1, d2, dtype=dtype)
    bad = [69, 70, 199, 259, n - 1]
    clean = ops.expert_mm(x, w, lens)
    dirty = x.clone()
    dirty[bad[0]], dirty[bad[1], 0], dirty[bad[2], -1] = NAN, INF, -INF
    dirty[sum(lens):] = NAN
    y = ops.expert_mm(dirty, w, lens)
    fine = torch.ones(n, dtype=torch.bool, device="cuda")
    fine[bad[:3]] = False
    assert torch.equal(y[fine], clean[fine])
    assert y[bad[0]].isnan().all() and not y[bad[1]].isfinite().any() \
        and not y[bad[2]].isfinite().any()
    X, W = dirty.clone().requires_grad_(), w.clone().requires_grad_()
    dw = torch.autograd.grad(ops.expert_mm(X, W, lens), W, dy)[0]
    assert dw[3].isfinite().all() and not dw[1].any()
    assert dw[0].isnan().all() and not dw[2, 0].isfinite().any()
    assert dw[2, 1:-1].isfinite().all()
    # a weight of one expert that is none
    w2 = w.clone()
    w2[2, 3, 4] = NAN
    y = ops.expert_mm(x, w2, lens)
    assert y[70:200, 4].isnan().all() and torch.equal(y[:70], clean[:70]) \
        and torch.equal(y[200:], clean[200:])
    assert torch.equal(y[70:200, 5:], clean[70:200, 5:])


def island(t, before):
    """The values of t, contiguous, `before` values into memory that is NaN around them."""
    sea = torch.full((before + t.numel() + 64,), NAN, device="cuda").to(t.dtype)
    it = sea[before:before + t.numel()].view(t.shape)
    it.copy_(t)
    return it


@pytest.mark.parametrize("before", [0, 1, 2, 5, 8])
@pytest.mark.parametrize("lens,behind", [([1], 0), ([3], 0), ([40, 0, 65], 0), ([40, 65], 6)])
@pytest.mark.parametrize("d1,d2", [(1, 1), (1, 2), (2, 3), (3, 130), (7, 8), (63, 9), (65, 127),
                                   (130, 129), (129, 64), (200, 33), (301, 602)])
def test_operands_are_read_to_their_ends_and_no_further(d1, d2, lens, behind, before):
    """Rows that end anywhere in 16 bytes, operands that begin and end anywhere in four."""
    g = gen(d1 * 1000 + d2)
    n, r = sum(lens) + behind, len(lens)
    x, dy = (island(rand(g, n, d, dtype=BF16), before) for d in (d1, d2))
    for turned in (False, True):
        if turned:
            w = island(rand(g, r, d2, d1, dtype=BF16), before).transpose(1, 2)
        else:
            w = island(rand(g, r, d1, d2, dtype=BF16), before)
        X, W = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = ops.expert_mm(X, W, lens)
        dx, dw = torch.autograd.grad(y, (X, W), dy)
        want, size = products(x, w, lens)
        check(y.detach(), want, (d1 + 64) * U * size, "y")
        want, size = products(dy, w.transpose(1, 2).contiguous(), lens)
        check(dx, want, (d2 + 64) * U * size, "dx")
        want, size = weight_gradients(x, dy, lens, r)
        check(dw, want, (max(lens) + 64) * U * size, "dw")
    qx, qw = ops.quantize_rows(x), ops.quantize_blocks(w)
    inner = island(qw.data.transpose(1, 2).contiguous(), before).transpose(1, 2)
    y = ops.scaled_mm(ops.Quantized(island(qx.data, before), qx.scale),
                      ops.Quantized(inner, qw.scale), lens, dtype=F32)
    want, size = products(values(qx, (1,)), values(qw, (1, 2)), lens)
    check(y, want, (d1 + 68) * U * size + cut(qx, qw, lens), "8 bits")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens,behind,d1,d2", [
    ([1], 0, 4096, 512), ([64], 0, 2048, 130), ([65], 0, 4104, 257), ([20], 44, 4103, 301),
    ([5, 0, 3], 9, 8200, 129), ([1, 2], 3, 1024, 4), ([300], 0, 1999, 64)])
def test_few_rows_of_long_inner_axes(lens, behind, d1, d2, dtype):
    """The inner axis in parts; a captured call has its own workspace."""
    g = gen(d1 + d2)
    n, r = sum(lens) + behind, len(lens)
    x, dy = rand(g, n, d1, dtype=dtype), rand(g, n, d1, dtype=dtype)
    w, v = rand(g, r, d1, d2, dtype=dtype), rand(g, r, d2, d1, dtype=dtype)
    qx, qw = ops.quantize_rows(x), ops.quantize_blocks(w)
    ids = torch.repeat_interleave(torch.arange(r + 1), torch.tensor(lens + [behind])).cuda()
    plan = ops.route_plan(ids, r)

    def run():
        return [ops.expert_mm(x, w, plan), ops.expert_mm(dy, v.transpose(1, 2), plan),
                ops.scaled_mm(qx, qw, plan, dtype=F32), ops.scaled_mm(qx, qw, plan, dtype=dtype)]

    y, z, eight, short = run()
    want, size = products(x, w, lens)
    check(y, want, (d1 + 64) * U * size, "y")
    want, size = products(dy, v.transpose(1, 2).contiguous(), lens)
    check(z, want, (d1 + 64) * U * size, "z")
    want, size = products(values(qx, (1,)), values(qw, (1, 2)), lens)
    check(eight, want, (d1 + 68) * U * size + cut(qx, qw, lens), "8 bits")
    assert torch.equal(short, eight.to(dtype))
    assert not any(t[sum(lens):].any() for t in (y, z, eight))
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(run())
    for seed in range(3):
        x.copy_(rand(gen(seed), n, d1, dtype=dtype))
        want = run()
        torch.cuda.synchronize()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_no_experts_and_no_inner_axis():
    x = torch.ones(5, 8, device="cuda", dtype=BF16)
    none = torch.ones(0, 8, 4, device="cuda", dtype=BF16)
    assert torch.equal(ops.expert_mm(x, none, []), torch.zeros_like(x[:, :4]))
    assert torch.equal(ops.scaled_mm(x, ops.quantize_blocks(none), []), torch.zeros_like(x[:, :4]))
    x, w = x[:, :0], torch.ones(2, 0, 4, device="cuda", dtype=BF16)
    for y in (ops.expert_mm(x, w, [2, 1]), ops.scaled_mm(x, ops.quantize_blocks(w), [2, 1]),
              ops.scaled_mm(x, ops.quantize_blocks(w[0]))):
        assert y.shape == (5, 4) and not y.any()
    X, W = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(ops.expert_mm(X, W, [2, 1]).sum(), (X, W))
    assert dx.shape == x.shape and dw.shape == w.shape


def test_subnormal_values_and_large_ones():
    """Products and sums keep float32's range: float16 subnormals count, and a result past
    the type's range is infinite."""
    x = torch.full((40, 64), 2.0 ** -24, device="cuda", dtype=F16)
    w = torch.full((1, 64, 16), 2.0 ** 10, device="cuda", dtype=F16)
    assert (ops.expert_mm(x, w, [40]) == 2.0 ** -8).all()
    w[:] = 60000.0
    assert (ops.expert_mm(torch.ones_like(x), w, [40]) == INF).all()
    x = torch.full((40, 64), 2.0 ** -130, device="cuda").to(BF16)
    w = torch.full((1, 64, 16), 2.0 ** 100, device="cuda").to(BF16)
    assert (ops.expert_mm(x, w, [40]) == 2.0 ** -24).all()


def test_views_containers_and_empty_calls():
    g = gen(3)
    x, w = rand(g, 50, 24, dtype=BF16), rand(g, 3, 24, 16, dtype=BF16)
    lens = [20, 0, 30]
    y = ops.expert_mm(x, w, lens)
    for lengths in (torch.tensor(lens), torch.tensor(lens).cuda(), torch.tensor(lens).float()):
        assert torch.equal(ops.expert_mm(x, w, lengths), y)
    # off a 16-byte boundary, other strides
    off = torch.empty(x.numel() + 1, dtype=BF16, device="cuda")[1:].view(50, 24).copy_(x)
    woff = torch.empty(w.numel() + 1, dtype=BF16, device="cuda")[1:].view(3, 24, 16).copy_(w)
    want, size = products(x, w, lens)
    for a, b in ((off, w), (x, woff), (off, woff), (x.t().contiguous().t(), w),
                 (x, w.permute(2, 1, 0).contiguous().permute(2, 1, 0))):
        check(ops.expert_mm(a, b, lens), want, (24 + 64) * U * size, "view")
    c = ops.expert_mm(x.cpu(), w.cpu(), lens)
    assert c.device.type == "cpu" and torch.equal(c, y.cpu())
    f = ops.expert_mm(x.float().cpu().numpy(), w.float().cpu().numpy(), lens)
    assert type(f).__name__ == "ndarray" and f.dtype == "float32"
    X, W = x.cpu().requires_grad_(), w.cpu().requires_grad_()
    ops.expert_mm(X, W, lens).float().sum().backward()
    assert X.grad.shape == x.shape and W.grad.device.type == "cpu" and not W.grad[1].any()
    for dtype in (BF16, F32):
        for n, r, d1, d2 in ((0, 3, 4, 5), (4, 0, 4, 5), (4, 2, 0, 5), (4, 2, 4, 0)):
            X = torch.ones(n, d1, device="cuda", dtype=dtype, requires_grad=True)
            W = torch.ones(r, d1, d2, device="cuda", dtype=dtype, requires_grad=True)
            y = ops.expert_mm(X, W, [0] * r)
            assert y.shape == (n, d2) and not y.any()
            dx, dw = torch.autograd.grad(y.sum(), (X, W))
            assert not dx.any() and not dw.any() and dw.shape == W.shape


def test_rows_past_32_bits():
    """More than 2**31 values of rows and of results; the last group behind them."""
    n, d = 2 ** 19 + 200, 4104
    x = torch.empty(n, d, dtype=BF16, device="cuda").fill_(1.0)
    g = gen(4)
    tail, w = rand(g, 150, d, dtype=BF16), rand(g, 2, d, d, dtype=BF16)
    x[-150:] = tail
    y = ops.expert_mm(x, w, [n - 150, 150])
    want, size = products(tail, w[1:], [150])
    check(y[-150:], want, (d + 64) * U * size, "tail")
    assert torch.equal(y[0], y[n - 151])
    dw = torch.empty(0)
    del y, dw
    W = w.clone().requires_grad_()
    dw = torch.autograd.grad(ops.expert_mm(x[:, :], W, [n - 150, 150]), W, x)[0]
    want, size = weight_gradients(tail, tail, [150], 1)
    check(dw[1:], want, (150 + 64) * U * size, "dw")


def test_differences():
    g = gen(5)
    x, w = rand(g, 12, 5, dtype=F64).requires_grad_(), rand(g, 3, 5, 4, dtype=F64).requires_grad_()
    assert torch.autograd.gradcheck(lambda a, b: ops.expert_mm(a, b, [4, 0, 7]), (x, w))


def test_some_gradients_and_versions():
    g = gen(6)
    x, w, dy = rand(g, 60, 40, dtype=BF16), rand(g, 2, 40, 24, dtype=BF16), rand(g, 60, 24,
                                                                                 dtype=BF16)
    X, W = x.clone().requires_grad_(), w.clone().requires_grad_()
    dx, dw = torch.autograd.grad(ops.expert_mm(X, W, [20, 35]), (X, W), dy)
    assert torch.equal(torch.autograd.grad(ops.expert_mm(X, w, [20, 35]), X, dy)[0], dx)
    assert torch.equal(torch.autograd.grad(ops.expert_mm(x, W, [20, 35]), W, dy)[0], dw)
    y = ops.expert_mm(X, W, [20, 35])
    with torch.no_grad():
        W.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_streams_and_graphs():
    """A layer on another stream, and captured: plans, products and gradients follow new
    rows and new routes on every replay."""
    g = gen(7)
    n, k, e, d1, d2 = 301, 2, 12, 136, 72
    x, w = rand(g, n, d1, dtype=BF16), rand(g, e, d1, d2, dtype=BF16)
    dy = rand(g, n * k, d2, dtype=BF16)
    ids = torch.randint(-1, e, (n, k), generator=g, device="cuda")
    q = ops.quantize_blocks(w)

    def run():
        plan = ops.route_plan(ids, e)
        X, W = x.detach().requires_grad_(), w.detach().requires_grad_()
        xs = ops.dispatch_rows(X, plan)
        y = ops.expert_mm(xs, W, plan)
        dx, dw = torch.autograd.grad(y, (X, W), dy)
        eight = ops.scaled_mm(ops.dispatch_rows(ops.quantize_rows(x), plan), q, plan)
        return [y.detach(), dx, dw, eight]

    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(4):
        h = gen(seed)
        x.copy_(rand(h, n, d1, dtype=BF16))
        ids.copy_(torch.randint(-1, e, (n, k), generator=h, device="cuda"))
        want = run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


# ---------------------------------------------------------------- 8 bits


def spread(scale, d, axis):
    return scale.double().repeat_interleave(128, axis).narrow(axis, 0, d)


def tops(q, axis, other=()):
    """The largest power of two in each eight neighbours along `axis` (2^-6 for e4m3's
    subnormals, 0 for zeros), times the scales."""
    v = q.data.double().abs()
    short = list(v.shape)
    short[axis] = -v.shape[axis] % 8
    v = torch.cat([v, v.new_zeros(short)], axis).unflatten(axis, (-1, 8)).amax(axis + 1)
    e = (torch.frexp(v).exponent - 1).clamp_min(-6)
    s = q.scale.double().repeat_interleave(16, axis).narrow(axis, 0, v.shape[axis])
    for a in other:
        s = s.repeat_interleave(128, a).narrow(a, 0, v.shape[a])
    return torch.where(v > 0, torch.ldexp(torch.ones_like(v), e), 0.0) * s


def cut(qx, qw, lens):
    """What the matrix cores leave out of products in 8 bits. They add the products of
    eight neighbours k in [8 j, 8 j + 8) cut off 13 binary places below the largest
    exponent ea + eb among them: 2^16 + 2^3 comes out whole, of 2^16 + 2^2 the second is
    lost. The largest, of two 4-bit mantissas, has 8 bits and stays whole; each of the
    seven others is off by less than 2^(ea + eb - 13). The exponent is at most the sum of
    the largest of either side: 7 * 2^-13 times the product of `tops`. (Of 650,000 random
    sums of 128, with zeros and subnormals among them, none was off by more than 4.1 of
    these 7 units, exponents taken product by product.)"""
    return 7 * 2.0 ** -13 * products(tops(qx, 1), tops(qw, 1, (2,)), lens)[0]


def values(q, axes):
    """What quantized values stand for, in float64."""
    s = q.scale
    for axis in axes:
        s = spread(s, q.data.shape[axis], axis)
    return q.data.double() * s


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_scaled_mm(shape, dtype):
    lens, behind, d1, d2 = SHAPES[shape]
    g = gen(shape + 100)
    n, r = sum(lens) + behind, len(lens)
    # blocks of unequal size
    x = rand(g, n, d1) * torch.exp(rand(g, d1))
    w = rand(g, r, d1, d2) * torch.exp(rand(g, d1, 1)) * d1 ** -0.5
    qx, qw = ops.quantize_rows(x), ops.quantize_blocks(w)
    y = ops.scaled_mm(qx, qw, lens, dtype=dtype)
    assert y.dtype == dtype
    want, size = products(values(qx, (1,)), values(qw, (1, 2)), lens)
    # besides: the product of the two scales and its product with a block's sum
    check(y, want, (d1 + 64 + 4) * U * size + cut(qx, qw, lens), "y")
    assert not y[sum(lens):].any()
    ids = torch.repeat_interleave(torch.arange(r + 1), torch.tensor(lens + [behind])).cuda()
    assert torch.equal(ops.scaled_mm(qx, qw, ops.route_plan(ids, r), dtype=dtype), y)
    if dtype == F32:  # rows that are quantised on the way; weights that lie the other way
        assert torch.equal(ops.scaled_mm(x, qw, lens), y)
        other = ops.Quantized(qw.data.contiguous(), qw.scale)
        assert torch.equal(ops.scaled_mm(qx, other, lens, dtype=F32), y)
    if len(lens) == 1 and not behind:
        one = ops.Quantized(qw.data[0], qw.scale[0])
        assert torch.equal(ops.scaled_mm(qx, one, dtype=dtype), y)
        assert torch.equal(ops.scaled_mm(qx, one, lens, dtype=dtype), y)


def test_scaled_mm_of_large_tiles():
    g = gen(8)
    lens, d1, d2 = [6000, 0, 5200], 2064, 1100
    x, w = rand(g, 11300, d1, dtype=BF16), rand(g, 3, d1, d2, dtype=BF16)
    qx, qw = ops.quantize_rows(x), ops.quantize_blocks(w)
    y = ops.scaled_mm(x, qw, lens)
    assert y.dtype == BF16 and torch.equal(ops.scaled_mm(qx, qw, lens), y)
    want, size = products(values(qx, (1,)), values(qw, (1, 2)), lens)
    check(y, want, (d1 + 68) * U * size + cut(qx, qw, lens), "y")
    half = ops.scaled_mm(x.half(), qw, lens)
    assert half.dtype == F16


@pytest.mark.parametrize("d1", [256, 250])
def test_scaled_mm_keeps_what_is_not_a_number_in_its_row(d1):
    g = gen(9)
    x, w = rand(g, 200, d1), rand(g, 2, d1, 40)
    qw = ops.quantize_blocks(w)
    clean = ops.scaled_mm(x, qw, [120, 60])
    x[119], x[120, 3], x[180:] = NAN, INF, NAN
    y = ops.scaled_mm(x, qw, [120, 60])
    fine = torch.ones(200, dtype=torch.bool, device="cuda")
    fine[119:121] = False
    assert torch.equal(y[fine], clean[fine]) and not y[180:].any()
    assert y[119].isnan().all() and y[120].isnan().all()


def test_refusals():
    x, w = torch.ones(6, 8, device="cuda"), torch.ones(2, 8, 4, device="cuda")
    plan = ops.route_plan(torch.zeros(6, 1, dtype=torch.int64, device="cuda"), 2)
    with pytest.raises(DGLError, match="plan is of 2 experts"):
        ops.expert_mm(x, w[:1], plan)
    with pytest.raises(DGLError, match="plan is of 6 entries"):
        ops.expert_mm(x[:5], w, plan)
    q, qw = ops.quantize_rows(x), ops.quantize_blocks(w)
    with pytest.raises(DGLError, match="no gradient"):
        ops.scaled_mm(x.clone().requires_grad_(), qw, plan)
    with pytest.raises(DGLError, match="no gradient"):
        ops.scaled_mm(q, ops.Quantized(qw.data, qw.scale.clone().requires_grad_()), plan)
    with pytest.raises(DGLError, match="no gradient"):
        ops.dispatch_rows(ops.Quantized(q.data, q.scale.clone().requires_grad_()), plan)


# ---------------------------------------------------------------- the layer


def test_dispatch_of_quantized_rows():
    g = gen(10)
    for d in (1, 7, 15, 16, 17, 100, 256, 1000):
        x = rand(g, 37, d)
        ids = torch.randint(-1, 5, (37, 3), generator=g, device="cuda")
        plan = ops.route_plan(ids, 5)
        q = ops.quantize_rows(x)
        out = ops.dispatch_rows(q, plan)
        assert isinstance(out, ops.Quantized) and out.data.dtype == F8
        assert torch.equal(out.data.float(), ops.dispatch_rows(q.data.float(), plan))
        assert torch.equal(out.scale, ops.dispatch_rows(q.scale, plan))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,d,e,k,f", [(37, 24, 5, 2, 40), (150, 136, 16, 4, 72), (3, 130, 8, 1, 64),
                                       (1, 256, 8, 2, 128)])
def test_a_layer_of_experts(dtype, n, d, e, k, f):
    """Norm with a residual, routing, the experts' products and the way back, and all
    gradients; in 8 bits the same from what was quantised. h is the half step of the
    rows' type, taken once for each rounding to it; each bound carries the one before
    it through the products."""
    g = gen(n)
    h = HALF_STEP[dtype]
    x, r = rand(g, n, d, dtype=dtype), rand(g, n, d, dtype=dtype)
    wn, w = rand(g, d), (rand(g, e, d, f, dtype=F64) * d ** -0.5).to(dtype)
    logits, dout = rand(g, n, e), rand(g, n, f, dtype=dtype)
    dtotal = rand(g, n, d, dtype=dtype)
    X, R, N, W, L = (t.clone().requires_grad_() for t in (x, r, wn, w, logits))
    y, total = ops.rms_norm(X, N, R)
    p, ids = ops.topk_route(L, k)
    plan = ops.route_plan(ids, e)
    out = ops.combine_rows(ops.expert_mm(ops.dispatch_rows(y, plan), W, plan), p, plan)
    dx, dr, dn, dw, dl = torch.autograd.grad((out, total), (X, R, N, W, L), (dout, dtotal))
    assert out.dtype == dx.dtype == dr.dtype == dw.dtype == dtype and torch.equal(dx, dr)

    t = x.double() + r.double()
    rs = 1.0 / (t.square().mean(1, keepdim=True) + 1e-6).sqrt()
    yd = t * rs * wn.double()
    e_y = (h + 80 * U) * yd.abs() + TINY[dtype]
    pd = torch.softmax(logits.double().gather(1, ids), 1)
    e_p = 60 * U * pd
    we = w.double()[ids]                                          # (n, k, d, f)
    ys = (yd[:, None, None, :] @ we)[:, :, 0]                     # (n, k, f)
    size = (yd.abs()[:, None, None, :] @ we.abs())[:, :, 0]
    e_ys = (1 + h) * ((e_y[:, None, None, :] @ we.abs())[:, :, 0] + (d + 64) * U * size) \
        + h * ys.abs() + TINY[dtype]
    want = (pd[:, :, None] * ys).sum(1)
    check(out.detach(), want, ((pd + e_p)[:, :, None] * e_ys + e_p[:, :, None] * ys.abs()
                               + (k + 2) * U * pd[:, :, None] * ys.abs()).sum(1), "out")

    # back: dys = p dout, rounded; dxs = dys W^T, rounded; dy the sum of a row's
    go = dout.double()
    dys = pd[:, :, None] * go[:, None, :]
    e_dys = (h + 70 * U) * dys.abs() + TINY[dtype]
    dxs = (dys[:, :, None, :] @ we.transpose(2, 3).contiguous())[:, :, 0]
    wt = we.abs().transpose(2, 3).contiguous()
    e_dxs = (1 + h) * ((e_dys[:, :, None, :] @ wt)[:, :, 0]
                       + (f + 64) * U * (dys.abs()[:, :, None, :] @ wt)[:, :, 0]) \
        + h * dxs.abs() + TINY[dtype]
    dy = dxs.sum(1)
    e_dy = (1 + h) * (e_dxs.sum(1) + (k + 2) * U * dxs.abs().sum(1)) + h * dy.abs() + TINY[dtype]
    dwd, e_dw = (torch.zeros(e, d, f, dtype=F64, device="cuda") for _ in range(2))
    for j in range(k):
        for i in range(n):
            c = ids[i, j]
            dwd[c] += yd[i, :, None] * dys[i, j]
            e_dw[c] += e_y[i, :, None] * dys[i, j].abs() \
                + (yd.abs() + e_y)[i, :, None] * e_dys[i, j] \
                + (n + 64) * U * yd.abs()[i, :, None] * dys[i, j].abs()
    check(dw, dwd, e_dw, "dw")
    xh = t * rs
    gw = dy * wn.double()
    e_g = e_dy * wn.double().abs() + 2 * U * gw.abs()
    q = (gw * xh).mean(1, keepdim=True)
    e_q = (e_g * xh.abs()).mean(1, keepdim=True) + 160 * U * (gw * xh).abs().mean(1, keepdim=True)
    dt = rs * (gw - xh * q) + dtotal.double()
    e_dt = rs * (e_g + xh.abs() * e_q) + 160 * U * (rs * (gw.abs() + xh.abs() * q.abs())
                                                     + dtotal.double().abs())
    check(dx, dt, e_dt, "dx")
    check(dn, (dy * xh).sum(0), (e_dy * xh.abs()).sum(0) + (n + 200) * U * (dy * xh).abs().sum(0),
          "dnorm")
    dp = (go[:, None, :] * ys).sum(2)
    e_dp = (go.abs()[:, None, :] * (e_ys + (f + 64) * U * ys.abs())).sum(2)
    dl_want = torch.zeros_like(logits, dtype=F64).scatter(
        1, ids, pd * (dp - (dp * pd).sum(1, keepdim=True)))
    scale = pd * (dp.abs() + (dp.abs() * pd).sum(1, keepdim=True))
    e_dl = torch.zeros_like(dl_want).scatter(
        1, ids, pd * (e_dp + (e_dp * pd).sum(1, keepdim=True)) * (1 + 100 * U) + 300 * U * scale)
    check(dl, dl_want, e_dl, "dlogits")

    # answering in 8 bits
    qw = ops.quantize_blocks(w)
    with torch.no_grad():
        qy, total8 = ops.rms_norm(X, N, R, quantize=True)
        rows = ops.scaled_mm(ops.dispatch_rows(qy, plan), qw, plan, dtype=dtype)
        out8 = ops.combine_rows(rows, p, plan)
    assert torch.equal(total8, total)
    a, b = values(qy, (1,)), values(qw, (1, 2))[ids]
    ys = (a[:, None, None, :] @ b)[:, :, 0]
    lost = 7 * 2.0 ** -13 * (tops(qy, 1)[:, None, None, :] @ tops(qw, 1, (2,))[ids])[:, :, 0]
    e_ys = h * ys.abs() + TINY[dtype] + (1 + h) * (
        lost + (d + 68) * U * (a.abs()[:, None, None, :] @ b.abs())[:, :, 0])
    want = (pd[:, :, None] * ys).sum(1)
    check(out8, want, ((pd + e_p)[:, :, None] * e_ys + e_p[:, :, None] * ys.abs()
                       + (k + 2) * U * pd[:, :, None] * ys.abs()).sum(1), "out8")

"""Root-mean-square norm and values in 8 bits on the GPU against plain float64, with
tolerances from the roundings each result passes through.

u is half a step of float32 (2^-24), half a step of the result's type is added for its
one rounding to it; e4m3 has steps of 2^(e - 3) for values of [2^e, 2^(e + 1)), none
below 2^-9."""

import threading

import pytest
import torch

import mojodgl.ops as ops
from mojodgl import DGLError

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
F8 = torch.float8_e4m3fn
HALF_STEP = {F32: 2.0 ** -24, F64: 2.0 ** -53, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -126, F64: 0.0, BF16: 2.0 ** -126, F16: 2.0 ** -24}
NAN, INF = float("nan"), float("inf")


def state(dtype):
    return F64 if dtype == F64 else F32


def within(got, want, limit, name):
    off = (got.double() - want).abs()
    assert got.shape == want.shape, name
    worst = int((off - limit).argmax()) if off.numel() else 0
    assert bool((off <= limit).all()), "{}: off by {} where {} is allowed".format(
        name, off.reshape(-1)[worst].item(), limit.expand_as(off).reshape(-1)[worst].item())


def check(got, want, bound, name):
    """|got - want| within `bound` (the error before the last rounding) and one
    rounding to got's type (for float16 subnormals: a step of 2^-24)."""
    h = HALF_STEP[got.dtype]
    within(got, want, bound * (1 + h) + want.abs() * h + TINY[got.dtype], name)


def rand(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=F64).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------- the norm


def reference(x, w, r, dy, dt, eps):
    """y, total, dx and dw in float64, and what the bounds need."""
    t = x.double() + (0.0 if r is None else r.double())
    w = torch.ones_like(t[..., :1, :]) if w is None else w.double()
    rs = 1.0 / (t.square().mean(-1, keepdim=True) + eps).sqrt()
    xh = t * rs
    out = {"t": t, "rs": rs, "xh": xh, "w": w, "y": xh * w}
    if dy is not None:
        g = dy.double() * w
        q = (g * xh).mean(-1, keepdim=True)
        out.update(g=g, q=q, dx=rs * (g - xh * q) + (0.0 if dt is None else dt.double()),
                   dw=(dy.double() * xh).reshape(-1, t.shape[-1]).sum(0))
    return out


def relative(d, u):
    """Relative error of rs: a sum of d squares in 64 or more partial sums of at most 32
    terms, joined pairwise (in order over d / 1024 terms of rows too wide for
    registers), passes 48 + d / 1024 roundings; t's own rounding, the quotient by d, eps
    and the root a few more."""
    return u * (48 + d / 1024 + 8)


def bounds(ref, dy, d, n, u):
    """Errors before the last rounding."""
    rel = relative(d, u)
    e_y = ref["y"].abs() * (rel + 4 * u)
    if dy is None:
        return e_y, None, None
    xh, g, q, rs = ref["xh"].abs(), ref["g"].abs(), ref["q"].abs(), ref["rs"]
    e_xh = xh * (rel + 4 * u)
    e_q = (g * e_xh + 2 * u * g * xh).mean(-1, keepdim=True) \
        + rel * (g * xh).mean(-1, keepdim=True)
    size = g + xh * q
    e_dx = rs * (2 * u * g + e_xh * q + xh * e_q + 4 * u * size) + rel * rs * size \
        + 4 * u * (ref["dx"].abs() + rs * size)
    rows = lambda z: z.reshape(-1, d).sum(0)  # noqa: E731
    # n rows in at most n / 256 + 64 + 64 additions one behind the other
    e_dw = rows(dy.double().abs() * e_xh) + (n / 64 + 160) * u * rows(dy.double().abs() * xh)
    return e_y, e_dx, e_dw


WIDTHS = [1, 2, 5, 7, 8, 15, 47, 63, 64, 100, 127, 128, 129, 255, 257, 511, 512, 602, 1023, 1024,
          1500, 2048, 2049, 4096, 4099, 8192, 8200, 16384, 16391]
TYPES = [(F32, F32, F32), (F64, F64, F64), (BF16, F32, F32), (BF16, BF16, BF16),
         (BF16, F32, BF16), (F16, F16, F32), (F16, F32, F16)]


@pytest.mark.parametrize("dtype,wdtype,rdtype", TYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_rms_norm(dtype, wdtype, rdtype, d):
    g = gen(d)
    n = 1 + (1777 * d) % 701 if d < 2048 else 5 + d % 7
    u = HALF_STEP[state(dtype)]
    x = (rand(g, n, d, dtype=F64) * (1 + torch.rand(d, generator=g, device="cuda"))).to(dtype)
    r, w = rand(g, n, d, dtype=rdtype), rand(g, d, dtype=wdtype)
    dy, dt = rand(g, n, d, dtype=dtype), rand(g, n, d, dtype=rdtype)
    # with the residual
    ref = reference(x, w, r, dy, dt, 1e-6)
    e_y, e_dx, e_dw = bounds(ref, dy, d, n, u)
    X, W, R = (t.clone().requires_grad_() for t in (x, w, r))
    y, total = ops.rms_norm(X, W, R)
    assert (y.dtype, total.dtype) == (dtype, rdtype)
    plain = ops.rms_norm(x, w, r)
    assert torch.equal(plain[0], y.detach()) and torch.equal(plain[1], total.detach())
    dx, dw, dr = torch.autograd.grad((y, total), (X, W, R), (dy, dt))
    assert (dx.dtype, dw.dtype, dr.dtype) == (dtype, wdtype, rdtype)
    check(y.detach(), ref["y"], e_y, "y")
    check(total.detach(), ref["t"], 2 * u * ref["t"].abs(), "total")
    check(dx, ref["dx"], e_dx, "dx")
    check(dr, ref["dx"], e_dx, "dresidual")
    check(dw, ref["dw"], e_dw, "dw")
    # and without
    ref = reference(x, w, None, dy, None, 0.1)
    e_y, e_dx, e_dw = bounds(ref, dy, d, n, u)
    X, W = (t.clone().requires_grad_() for t in (x, w))
    y = ops.rms_norm(X, W, eps=0.1)
    dx, dw = torch.autograd.grad(y, (X, W), dy)
    check(y.detach(), ref["y"], e_y, "y alone")
    check(dx, ref["dx"], e_dx, "dx alone")
    check(dw, ref["dw"], e_dw, "dw alone")


@pytest.mark.parametrize("d", [33, 512, 3000, 20000])
@pytest.mark.parametrize("rdtype", [BF16, F32])
@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)])
def test_some_gradients(need, rdtype, d):
    g = gen(3)
    ops_in = rand(g, 70, d, dtype=BF16), rand(g, d), rand(g, 70, d, dtype=rdtype)
    dy, dt = rand(g, 70, d, dtype=BF16), rand(g, 70, d, dtype=rdtype)
    leaves = [t.clone().requires_grad_() for t in ops_in]
    for outs in ((0, 1), (0,), (1,)):
        def grads(which):
            some = [t.detach().requires_grad_(bool(k)) for t, k in zip(ops_in, which)]
            res = ops.rms_norm(*some)
            return torch.autograd.grad([res[i] for i in outs], [t for t in some if t.requires_grad],
                                       [(dy, dt)[i] for i in outs], allow_unused=True)

        whole = grads((1, 1, 1))
        if outs == (1,) and need == (0, 1, 0):
            continue  # total does not depend on the weight alone
        for a, b in zip(grads(need), [t for t, k in zip(whole, need) if k]):
            assert torch.equal(a, b)
    if rdtype == BF16:
        assert whole[0].data_ptr() == whole[2].data_ptr() or torch.equal(whole[0], whole[2])
    # total's gradient alone passes both ways unchanged
    assert torch.equal(whole[2], dt) and not whole[1].any()
    del leaves


def test_shapes_layouts_and_containers():
    g = gen(4)
    x, r = rand(g, 3, 5, 48, dtype=BF16), rand(g, 3, 5, 48, dtype=BF16)
    y, total = ops.rms_norm(x, None, r)
    assert y.shape == total.shape == (3, 5, 48)
    flat = ops.rms_norm(x.reshape(15, 48), None, r.reshape(15, 48))
    assert torch.equal(y.reshape(15, 48), flat[0]) and torch.equal(total.reshape(15, 48), flat[1])
    turned = ops.rms_norm(x.transpose(0, 1), None, r.transpose(0, 1).contiguous())
    assert torch.equal(turned[0], y.transpose(0, 1))
    # one element off a 16-byte boundary
    off = torch.empty(x.numel() + 1, dtype=BF16, device="cuda")[1:].view(3, 5, 48).copy_(x)
    assert torch.equal(ops.rms_norm(off, None, r)[0], y)
    # numpy and CPU tensors come back as they are
    a = ops.rms_norm(x.float().cpu().numpy(), residual=r.float().cpu().numpy())
    assert type(a[0]).__name__ == type(a[1]).__name__ == "ndarray" and a[0].dtype == "float32"
    b = ops.rms_norm(x.cpu(), residual=r.cpu())
    assert b[0].device.type == "cpu" and torch.equal(b[0], y.cpu()) \
        and torch.equal(b[1], total.cpu())
    X, R = x.cpu().requires_grad_(), r.cpu().requires_grad_()
    y, total = ops.rms_norm(X, None, R)
    (y.float().sum() + total.float().sum()).backward()
    assert X.grad.device.type == "cpu" and torch.equal(X.grad, R.grad)
    for shape in ((0, 16), (4, 0), (0, 0)):
        y, total = ops.rms_norm(torch.zeros(shape, device="cuda"), None,
                                torch.zeros(shape, device="cuda"))
        assert y.shape == total.shape == shape
        W = torch.ones(shape[1], device="cuda", requires_grad=True)
        ops.rms_norm(torch.zeros(shape, device="cuda"), W).sum().backward()
        assert not W.grad.any()
    # float64 anywhere makes the rows float64; a float32 residual beside 16 bits stays
    one = torch.ones(2, 4, device="cuda")
    assert ops.rms_norm(one, one[0].double())[0].dtype == F64
    assert [t.dtype for t in ops.rms_norm(one, None, one.double())] == [F64, F64]
    assert [t.dtype for t in ops.rms_norm(one.half(), None, one.bfloat16())] == [F16, F32]


def test_rows_that_are_not_numbers_stay_alone():
    x = torch.ones(6, 300, device="cuda")
    x[1, 7], x[2, 8], x[3] = NAN, INF, 0.0
    y = ops.rms_norm(x)
    assert y[1].isnan().all() and y[2, 8].isnan() and (y[2, :8] == 0).all()
    assert (y[3] == 0).all() and torch.equal(y[0], y[4]) and y[0].isfinite().all()
    assert ops.rms_norm(x, eps=0.0)[3].isnan().all()


def test_differences():
    g = gen(6)
    x, w, r = (rand(g, *s, dtype=F64).requires_grad_() for s in ((4, 9), (9,), (4, 9)))
    assert torch.autograd.gradcheck(lambda *a: ops.rms_norm(*a, eps=0.01), (x, w, r))


def test_what_is_written_over_is_seen():
    """The backward pass reads a float32 sum, or 16-bit rows and residuals."""
    for dtype in (F32, BF16):
        x = torch.rand(3, 8, device="cuda").to(dtype).requires_grad_()
        r = torch.rand(3, 8, device="cuda").to(dtype)
        for saved in (0, 1):
            y, total = ops.rms_norm(x, None, r)
            with torch.no_grad():
                (total if saved else r).add_(1.0)
            if saved == (dtype == F32):
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    y.sum().backward()
            else:
                y.sum().backward()


def test_many_rows_past_32_bits():
    """More than 2**31 values: the last rows lie behind 32-bit offsets."""
    n, d = 2 ** 21 + 3, 1040
    x = torch.empty(n, d, dtype=BF16, device="cuda").fill_(2.0)
    tail = rand(gen(1), 5, d, dtype=BF16)
    x[-5:] = tail
    assert torch.equal(ops.rms_norm(x)[-5:], ops.rms_norm(tail))
    q, few = ops.rms_norm(x, quantize=True), ops.rms_norm(tail, quantize=True)
    assert torch.equal(q.data[-5:].view(torch.uint8), few.data.view(torch.uint8))
    assert torch.equal(q.scale[-5:], few.scale)
    q, few = ops.quantize_rows(x), ops.quantize_rows(tail)
    assert torch.equal(q.data[-5:].view(torch.uint8), few.data.view(torch.uint8))


# ---------------------------------------------------------------- 8 bits


def e4m3_half_step(v):
    e = torch.frexp(v.abs().clamp_min(2.0 ** -6)).exponent - 1
    return torch.ldexp(torch.ones_like(v), e - 4)


def spread(scale, d, axis):
    return scale.double().repeat_interleave(128, axis).narrow(axis, 0, d)


def check_values(data, scale, want, e_want, axes, name):
    """Each value within half a step of e4m3 of what it stands for (float32 quotients
    are off by 2^-23 of it besides), its scale within its own rounding."""
    tops = want.abs()
    for axis in axes:
        short = -tops.shape[axis] % 128
        pad = list(tops.shape)
        pad[axis] = short
        tops = torch.cat([tops, tops.new_zeros(pad)], axis)
        tops = tops.unflatten(axis, (-1, 128)).amax(axis + 1 if axis >= 0 else axis)
    assert scale.dtype == F32 and scale.shape == tops.shape, name
    top = (tops / 448).clamp_min(2.0 ** -126)
    e_rel = e_want + 2.0 ** -23
    within(scale, top, top * e_rel, name + " scales")
    s = scale.double()
    for axis in axes:
        s = spread(s, want.shape[axis], axis)
    v = want / s
    assert data.dtype == F8, name
    within(data.float(), v, e4m3_half_step(v) * (1 + 2.0 ** -20) + v.abs() * e_rel, name)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("d", WIDTHS)
def test_quantize_rows(dtype, d):
    g = gen(d + 1)
    n = 1 + (1777 * d) % 701 if d < 2048 else 5 + d % 7
    x = (rand(g, n, d, dtype=F64) * torch.exp(2 * rand(g, n, d, dtype=F64))).clamp(-6e4, 6e4)
    x = x.to(dtype)
    x[0] = 0.0
    q = ops.quantize_rows(x)
    assert q.data.shape == x.shape
    check_values(q.data, q.scale, x.double(), 0.0, (-1,), "rows")
    assert (q.data[0].float() == 0).all() and (q.scale[0] == 2.0 ** -126).all()


@pytest.mark.parametrize("dtype,wdtype,rdtype", [t for t in TYPES if t[0] != F64])
@pytest.mark.parametrize("d", WIDTHS)
def test_rms_norm_in_8_bits(dtype, wdtype, rdtype, d):
    g = gen(d + 2)
    n = 1 + (1777 * d) % 401 if d < 2048 else 5 + d % 7
    x, r, w = rand(g, n, d, dtype=dtype), rand(g, n, d, dtype=rdtype), rand(g, d, dtype=wdtype)
    ref = reference(x, w, r, None, None, 1e-6)
    (q, scale), total = ops.rms_norm(x, w, r, quantize=True)
    y, total_of_y = ops.rms_norm(x, w, r)
    assert torch.equal(total, total_of_y)
    check_values(q, scale, ref["y"], relative(d, HALF_STEP[F32]) + 4 * HALF_STEP[F32], (-1,), "y")
    if dtype == F32:  # where y is not rounded in between, it is quantize_rows of it
        again = ops.quantize_rows(y)
        assert torch.equal(again.data.view(torch.uint8), q.view(torch.uint8))
        assert torch.equal(again.scale, scale)
    alone = ops.rms_norm(x, w, quantize=True)
    assert isinstance(alone, ops.Quantized) and alone.data.shape == x.shape


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("r,d1,d2", [(1, 1, 1), (3, 128, 128), (2, 129, 127), (5, 7, 300),
                                     (2, 300, 9), (1, 1000, 602), (4, 256, 384), (70, 33, 65)])
def test_quantize_blocks(dtype, r, d1, d2):
    g = gen(d1 + d2)
    w = rand(g, r, d1, d2, dtype=dtype)
    q = ops.quantize_blocks(w)
    assert q.data.shape == w.shape and q.data.transpose(1, 2).is_contiguous()
    check_values(q.data, q.scale, w.double(), 0.0, (-2, -1), "blocks")
    turned = ops.quantize_blocks(w.transpose(1, 2).contiguous().transpose(1, 2))
    for a, b in zip(q, turned):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    one = ops.quantize_blocks(w[0])
    assert one.data.shape == (d1, d2) and torch.equal(one.scale, q.scale[0])


def test_ties_and_borders():
    """A block of scale 1: every e4m3 value, the middles between neighbours (to the even
    one) and the floats beside the middles."""
    codes = torch.arange(127, dtype=torch.uint8, device="cuda").view(F8).float()  # 0 .. 448
    mid = (codes[:-1] + codes[1:]) / 2
    want_mid = torch.where(torch.arange(126, device="cuda") % 2 == 0, codes[:-1], codes[1:])
    lo = torch.nextafter(mid, torch.zeros_like(mid))
    hi = torch.nextafter(mid, torch.full_like(mid, 1e9))
    x = torch.stack([codes, *(torch.cat([t, t.new_full((1,), 448.0)]) for t in (mid, lo, hi))])
    x = torch.cat([x, -x])
    q = ops.quantize_rows(x)
    assert (q.scale == 1).all()
    want = torch.stack([codes, *(torch.cat([t, codes[-1:]]) for t in (want_mid, codes[:-1],
                                                                     codes[1:]))])
    assert torch.equal(q.data.float(), torch.cat([want, -want]))


def test_small_and_large_scales():
    """Blocks from the least subnormals to the largest floats: scales at their least, and
    quotients right where reciprocals would not be normal."""
    g = gen(9)
    base = rand(g, 60, 128).abs().clamp(0.01, 4.0) * torch.sign(rand(g, 60, 128))
    e = torch.linspace(-148, 125, 60, device="cuda").round().double()
    x = (base.double() * torch.exp2(e)[:, None]).float()
    q = ops.quantize_rows(x)
    top = (x.double().abs().amax(1, keepdim=True) / 448).clamp_min(2.0 ** -126)
    # a subnormal's quotient by 448 is cut off by half the least subnormal at most
    within(q.scale, top, top * 2.0 ** -23, "scales")
    v = x.double() / q.scale.double()
    within(q.data.float(), v, e4m3_half_step(v) * (1 + 2.0 ** -20) + v.abs() * 2.0 ** -23, "values")


def test_not_numbers_in_8_bits():
    x = torch.ones(3, 300, device="cuda")
    x[0, 3], x[1, 130], x[2, 299] = NAN, INF, -INF
    for data, scale in (ops.quantize_rows(x), ops.quantize_rows(x.bfloat16())):
        back = data.float() * spread(scale, 300, 1)
        assert back[0, 3].isnan() and (back[0, :3] - 1).abs().max() < 2.0 ** -4
        assert torch.equal(scale[0], scale[0, :1].expand(3)) and scale[1, 1] == INF
        assert back[1, 128:256].isnan().all() and back[1, :128].isfinite().all()
        assert back[2, 256:].isnan().all() and back[2, :256].isfinite().all()
    w = torch.ones(200, 200, device="cuda")
    w[3, 150] = NAN
    data, scale = ops.quantize_blocks(w)
    assert scale.isfinite().all() and data.float().isnan().sum() == 1 and data[3, 150].isnan()


def test_refusals():
    x = torch.ones(4, 8, device="cuda")
    with pytest.raises(DGLError, match="float64"):
        ops.rms_norm(x.double(), quantize=True)
    with pytest.raises(DGLError, match="no gradient"):
        ops.rms_norm(x.clone().requires_grad_(), quantize=True)
    with pytest.raises(DGLError, match="no gradient"):
        ops.quantize_rows(x.clone().requires_grad_())
    with torch.no_grad():
        ops.quantize_rows(x.clone().requires_grad_())


def test_streams_and_graphs():
    """On another stream behind its producer, and captured, replayed with new inputs."""
    g = gen(11)
    x, r, w = rand(g, 333, 1000, dtype=BF16), rand(g, 333, 1000), rand(g, 1000)

    def run(x, r, w):
        (data, scale), total = ops.rms_norm(x, w, r, quantize=True)
        X, W = x.detach().requires_grad_(), w.detach().requires_grad_()
        y, t2 = ops.rms_norm(X, W, r)
        dx, dw = torch.autograd.grad((y, t2), (X, W), (x, r))
        q = ops.quantize_rows(y.detach())
        return [data.view(torch.uint8), scale, total, y.detach(), dx, dw, q.data.view(torch.uint8)]

    want = run(x, r, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run((x.float() * 2).bfloat16() / 2, r, w)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, r, w)
    for seed in range(3):
        x.copy_(rand(gen(seed), 333, 1000, dtype=BF16))
        want = run(x, r, w)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_threads():
    g = gen(12)
    xs = [rand(g, 257, 700 + i, dtype=BF16) for i in range(4)]
    want = [ops.rms_norm(x, quantize=True) for x in xs]
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                q = ops.rms_norm(xs[i], quantize=True)
            torch.cuda.current_stream().synchronize()
        if not all(torch.equal(a.view(torch.uint8), b.view(torch.uint8))
                   for a, b in zip(q, want[i])):
            bad.append(i)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad

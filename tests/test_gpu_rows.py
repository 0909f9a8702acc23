"""Layer norm and the segment scan on the GPU against plain float64, with tolerances
from the roundings each result passes through.

u is half a step of float32 (2^-24), half a step of the result's type is added for
its one rounding to it. Sizes are those where lanes, vectors, strips and chunks
begin and end; lengths from none to several chunks."""

import threading

import numpy as np
import pytest
import torch

import mojodgl as dgl
import mojodgl.ops as ops
from mojodgl import DGLError

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
HALF_STEP = {F32: 2.0 ** -24, F64: 2.0 ** -53, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -126, F64: 0.0, BF16: 2.0 ** -126, F16: 2.0 ** -24}


def state(dtype):
    return F64 if dtype == F64 else F32


def check(got, want, bound, name):
    """|got - want| within `bound` (float64, the error before the last rounding) and
    one rounding to got's type (for float16 subnormals: a step of 2^-24)."""
    assert got.shape == want.shape, name
    limit = bound * (1 + HALF_STEP[got.dtype]) + want.abs() * HALF_STEP[got.dtype] \
        + TINY[got.dtype]
    off = (got.double() - want).abs()
    worst = int((off - limit).argmax()) if off.numel() else 0
    assert bool((off <= limit).all()), "{}: off by {} where {} is allowed".format(
        name, off.reshape(-1)[worst].item(), limit.expand_as(off).reshape(-1)[worst].item())


def rand(gen, *shape, dtype=F32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=F64).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---------------------------------------------------------------- layer norm


def norm_reference(x, w, b, dy, eps):
    x, w, b, dy = (None if t is None else t.double() for t in (x, w, b, dy))
    d = x.shape[-1]
    c = x - x.mean(-1, keepdim=True)
    r = 1.0 / (c.square().mean(-1, keepdim=True) + eps).sqrt()
    xh = c * r
    y = xh * (1.0 if w is None else w) + (0.0 if b is None else b)
    g = dy * (1.0 if w is None else w)
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    rows = (-1, d)
    return (xh, r, y, dx, (dy * xh).reshape(rows).sum(0), dy.reshape(rows).sum(0))


def norm_bounds(x, w, dy, xh, r, n, d, u):
    """Errors before the last rounding. A sum of d terms in 64 or more partial sums
    of at most 32 terms, joined pairwise, passes s = 32 + 16 roundings at most (in
    order over at most d / 1024 terms beyond 32,768 columns). mean: s u mean|x|.
    x - mean: that and one rounding. The variance: twice the relative error of the
    centred values (in the mean square) and s u. xh then is off by the centred
    value's error times r and by |xh| (s + 8) u."""
    s = 48 + d / 1024
    x, dy = x.double(), dy.double()
    centre = u * (s * x.abs().mean(-1, keepdim=True) + 2 * x.abs()) * r
    mean_centre = centre.square().mean(-1, keepdim=True).sqrt()
    e_xh = centre + xh.abs() * (u * (s + 8) + 2 * mean_centre)
    gw = 1.0 if w is None else w.double().abs()
    g = dy.abs() * gw
    e_y = e_xh * gw + 4 * u * (xh.abs() * gw)
    e_g = 2 * u * g
    mean_g = g.mean(-1, keepdim=True)
    mean_q = (g * xh.abs()).mean(-1, keepdim=True)
    e_q = (g * e_xh + e_g * xh.abs()).mean(-1, keepdim=True) + s * u * mean_q
    inner = e_g + s * u * mean_g + e_xh * mean_q + xh.abs() * e_q \
        + 4 * u * (g + mean_g + xh.abs() * mean_q)
    rel_r = u * (s + 8) + 2 * mean_centre
    e_dx = r * inner + rel_r * r * (g + mean_g + xh.abs() * mean_q)
    # n rows in at most n / 256 + 64 + 64 additions one behind the other
    t = n / 64 + 160
    flat = lambda z: z.expand_as(dy).reshape(-1, d).sum(0)  # noqa: E731
    e_dw = flat(dy.abs() * e_xh) + t * u * flat(dy.abs() * xh.abs())
    e_db = t * u * flat(dy.abs())
    return e_y, e_dx, e_dw, e_db


NORM_WIDTHS = [1, 2, 3, 4, 5, 7, 8, 15, 16, 31, 47, 63, 64, 100, 127, 128, 255, 256, 257, 511,
               512, 513, 602, 1023, 1024, 1500, 2048, 2049, 4096, 4099, 8192, 8200, 16384, 16391]


@pytest.mark.parametrize("dtype,wdtype", [(F32, F32), (F64, F64), (BF16, F32), (BF16, BF16),
                                          (F16, F32), (F16, F16)])
@pytest.mark.parametrize("d", NORM_WIDTHS)
def test_layer_norm(dtype, wdtype, d):
    g = gen(d)
    n = 1 + (1777 * d) % 701 if d < 2048 else 5 + d % 7
    x = (rand(g, n, d, dtype=F64) * (1 + torch.rand(d, generator=g, device="cuda")) + 1.5).to(dtype)
    w, b = rand(g, d, dtype=wdtype), rand(g, d, dtype=wdtype)
    dy = rand(g, n, d, dtype=dtype)
    xh, r, y0, dx0, dw0, db0 = norm_reference(x, w, b, dy, 1e-5)
    e_y, e_dx, e_dw, e_db = norm_bounds(x, w, dy, xh, r, n, d, HALF_STEP[state(dtype)])
    e_y = e_y + 2 * HALF_STEP[state(dtype)] * b.double().abs()
    X, W, B = (t.clone().requires_grad_() for t in (x, w, b))
    y = ops.layer_norm(X, W, B)
    assert y.dtype == dtype and torch.equal(ops.layer_norm(x, w, b), y.detach())
    dx, dw, db = torch.autograd.grad(y, (X, W, B), dy)
    assert (dx.dtype, dw.dtype, db.dtype) == (dtype, wdtype, wdtype)
    check(y.detach(), y0, e_y, "y")
    check(dx, dx0, e_dx, "dx")
    check(dw, dw0, e_dw, "dw")
    check(db, db0, e_db, "db")


@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1)])
@pytest.mark.parametrize("d", [33, 512, 20000])
def test_layer_norm_some_gradients(need, d):
    g = gen(3)
    x, w, b, dy = rand(g, 70, d), rand(g, d), rand(g, d), rand(g, 70, d)
    X, W, B = (t.clone().requires_grad_() for t in (x, w, b))
    whole = torch.autograd.grad(ops.layer_norm(X, W, B), (X, W, B), dy)
    some = [t.clone().requires_grad_(bool(k)) for t, k in zip((x, w, b), need)]
    got = torch.autograd.grad(ops.layer_norm(*some), [t for t in some if t.requires_grad], dy)
    for a, b_ in zip(got, [t for t, k in zip(whole, need) if k]):
        assert torch.equal(a, b_)


def test_layer_norm_without_weights_and_other_shapes():
    g = gen(4)
    x = rand(g, 3, 0 + 5, 7, 24)
    dy = rand(g, 3, 5, 7, 24)
    xh, r, y0, dx0, _, _ = norm_reference(x, None, None, dy, 0.5)
    e_y, e_dx, _, _ = norm_bounds(x, None, dy, xh, r, 105, 24, 2.0 ** -24)
    X = x.clone().requires_grad_()
    y = ops.layer_norm(X, eps=0.5)
    check(y.detach(), y0, e_y, "y")
    check(torch.autograd.grad(y, X, dy)[0], dx0, e_dx, "dx")
    b = rand(g, 24)
    check(ops.layer_norm(x, bias=b, eps=0.5), y0 + b.double(), e_y + 2.0 ** -22, "bias alone")
    # no rows, no columns, one row without an axis in front
    w = torch.ones(6, device="cuda", requires_grad=True)
    e = torch.zeros(0, 6, device="cuda", requires_grad=True)
    de, dw = torch.autograd.grad(ops.layer_norm(e, w).sum(), (e, w))
    assert de.shape == (0, 6) and torch.equal(dw, torch.zeros(6, device="cuda"))
    z = torch.zeros(4, 0, device="cuda", requires_grad=True)
    assert ops.layer_norm(z).shape == (4, 0)
    assert torch.autograd.grad(ops.layer_norm(z).sum(), z)[0].shape == (4, 0)
    assert torch.equal(ops.layer_norm(x[0, 0, 0], eps=0.5), ops.layer_norm(x, eps=0.5)[0, 0, 0])
    # a constant row has no spread: eps alone
    assert torch.equal(ops.layer_norm(torch.full((2, 100), 3.0, device="cuda"), bias=None),
                       torch.zeros(2, 100, device="cuda"))


def test_layer_norm_containers_and_types():
    rng = np.random.default_rng(0)
    x, w = rng.standard_normal((5, 9)), rng.standard_normal(9)
    got = ops.layer_norm(x, w)
    assert isinstance(got, np.ndarray) and got.dtype == np.float64
    xc = x - x.mean(1, keepdims=True)
    np.testing.assert_allclose(got, xc / np.sqrt((xc ** 2).mean(1, keepdims=True) + 1e-5) * w,
                               rtol=1e-13, atol=1e-14)
    assert ops.layer_norm(x.astype(np.float16)).dtype == np.float16
    assert ops.layer_norm(x.astype(np.float32), w).dtype == np.float64  # float64 weights
    h = torch.from_numpy(x).to(BF16)  # a CPU tensor: results and gradients on the CPU
    H = h.clone().requires_grad_()
    y = ops.layer_norm(H, torch.from_numpy(w).float())
    assert y.device.type == "cpu" and y.dtype == BF16
    assert torch.autograd.grad(y.sum(), H)[0].device.type == "cpu"
    # weights of two types meet in float32
    y = ops.layer_norm(h.cuda(), torch.ones(9, device="cuda", dtype=BF16),
                       torch.zeros(9, device="cuda"))
    assert torch.equal(y, ops.layer_norm(h.cuda()))


def test_layer_norm_strides_and_alignment():
    g = gen(5)
    wide = rand(g, 40, 131, dtype=BF16)
    for x in (wide[:, 1:], wide[:, 3:67], wide.t(), wide[::2], wide[0].expand(6, 131)):
        assert torch.equal(ops.layer_norm(x), ops.layer_norm(x.contiguous()))
    # rows that are contiguous but start at odd addresses
    for off in (1, 3, 5):
        flat = rand(g, off + 10 * 72, dtype=F16)
        x = flat[off:].view(10, 72)
        w = rand(g, off + 72)[off:]
        assert torch.equal(ops.layer_norm(x, w), ops.layer_norm(x.clone(), w.clone()))


def test_layer_norm_infinities_stay_in_their_rows():
    x = torch.randn(64, 130, device="cuda")
    want = ops.layer_norm(x)
    y = x.clone()
    y[3, 5], y[10, 0], y[40, 129] = float("inf"), float("nan"), -float("inf")
    got = ops.layer_norm(y)
    rest = [i for i in range(64) if i not in (3, 10, 40)]
    assert torch.equal(got[rest], want[rest]) and bool(got[[3, 10, 40]].isnan().all())


def test_layer_norm_large_means():
    """The variance is summed around the mean: a mean of 1,000 standard deviations
    costs the rows' own rounding, not the square of it."""
    g = gen(6)
    x = rand(g, 50, 777) + 1000.0
    xh, r, y0, _, _, _ = norm_reference(x, None, None, torch.zeros_like(x), 1e-5)
    e_y, _, _, _ = norm_bounds(x, None, torch.zeros_like(x), xh, r, 50, 777, 2.0 ** -24)
    check(ops.layer_norm(x), y0, e_y, "y")
    assert bool((ops.layer_norm(x).double() - y0).abs().max() < 2e-3)


# ---------------------------------------------------------------- the scan


def scan_reference(lens, a, v, init, dh, dl):
    """Row by row in float64, and for each result a bound on a float32 evaluation: a
    term that passes t rows takes part in 2 t roundings, and in at most 40 more where
    chunks' and strips' maps are composed (`slack`)."""
    u = HALF_STEP[state(v.dtype)]
    a, v, dh = a.double().cpu(), v.double().cpu(), dh.double().cpu()
    n, d = a.shape
    s = len(lens)
    init = torch.zeros(s, d, dtype=F64) if init is None else init.double().cpu()
    dl = torch.zeros(s, d, dtype=F64) if dl is None else dl.double().cpu()
    h, eh, da, ea, dv, ev = (torch.zeros(n, d, dtype=F64) for _ in range(6))
    last, elast, di, edi = (torch.zeros(s, d, dtype=F64) for _ in range(4))
    slack = 40 * u
    at = 0
    for k, m in enumerate(lens):
        cur, size, e = init[k].clone(), init[k].abs(), torch.zeros(d, dtype=F64)
        before, ebefore = [], []
        for t in range(at, at + m):
            before.append(cur)
            ebefore.append(e + slack * size)
            size = a[t].abs() * size + v[t].abs()
            e = a[t].abs() * e + 2 * u * size
            cur = a[t] * cur + v[t]
            h[t], eh[t] = cur, e + slack * size
        last[k], elast[k] = cur, e + slack * size
        c, size, e = dl[k].clone(), dl[k].abs(), torch.zeros(d, dtype=F64)
        for t in range(at + m - 1, at - 1, -1):
            g, size = dh[t] + c, dh[t].abs() + size
            e = e + u * size
            dv[t], ev[t] = g, e + slack * size
            da[t] = g * before[t - at]
            ea[t] = (e + slack * size) * (before[t - at].abs() + ebefore[t - at]) \
                + g.abs() * ebefore[t - at] + 2 * u * da[t].abs()
            c, size, e = a[t] * g, a[t].abs() * size, a[t].abs() * (e + u * size)
        di[k], edi[k] = c, e + slack * size
        at += m
    return [(x.cuda(), y.cuda()) for x, y in ((h, eh), (last, elast), (da, ea), (dv, ev),
                                              (di, edi))]


def scan_inputs(seed, lens, d, dtype, gdtype, low=0.0):
    g = gen(seed)
    n, s = sum(lens), len(lens)
    a = (low + (1 - low) * torch.rand(n, d, generator=g, device="cuda", dtype=F64)).to(gdtype)
    st = state(dtype)
    return (a, rand(g, n, d, dtype=dtype), rand(g, s, d, dtype=st), rand(g, n, d, dtype=dtype),
            rand(g, s, d, dtype=st))


SCAN_LENS = [[1], [2, 0, 3], [0, 0, 5], [16], [15, 1, 17], [16, 16, 0], [128], [127, 1, 1],
             [129], [5, 300, 0, 0, 70], [1000], [31] * 9 + [0], [0, 513, 2, 255, 0]]
SCAN_TYPES = [(F32, F32), (F64, F64), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]


@pytest.mark.parametrize("dtype,gdtype", SCAN_TYPES)
@pytest.mark.parametrize("d", [1, 2, 3, 7, 16, 33, 100, 130, 257])
def test_scan(dtype, gdtype, d):
    for k, lens in enumerate(SCAN_LENS):
        a, v, init, dh, dl = scan_inputs(10 * d + k, lens, d, dtype, gdtype,
                                         low=(0.0, 0.9)[k % 2])
        A, V, I = (t.clone().requires_grad_() for t in (a, v, init))  # noqa: E741
        h, last = ops.segment_scan(lens, A, V, I, return_state=True)
        assert h.dtype == dtype and last.dtype == state(dtype)
        grads = torch.autograd.grad((h, last), (A, V, I), (dh, dl))
        got = [h.detach(), last.detach()] + list(grads)
        for name, x, (want, bound) in zip(("h", "last", "dgate", "dvalue", "dinitial"), got,
                                          scan_reference(lens, a, v, init, dh, dl)):
            check(x, want, bound, "{} {}".format(name, lens))
        # no gradient asked for, no states: the same h
        assert torch.equal(ops.segment_scan(lens, a, v, init), h.detach())


@pytest.mark.parametrize("lens,d", [([3000], 5), ([2500, 0, 1, 1400], 66), ([4096, 37], 129)])
def test_scan_over_many_chunks(lens, d):
    """Chains of chunks that look back over each other, with memories of thousands
    of rows."""
    a, v, init, dh, dl = scan_inputs(len(lens), lens, d, F32, F32, low=0.999)
    A, V, I = (t.clone().requires_grad_() for t in (a, v, init))  # noqa: E741
    h, last = ops.segment_scan(torch.tensor(lens, device="cuda"), A, V, I, return_state=True)
    got = [h.detach(), last.detach()] + list(torch.autograd.grad((h, last), (A, V, I), (dh, dl)))
    for name, x, (want, bound) in zip(("h", "last", "dgate", "dvalue", "dinitial"), got,
                                      scan_reference(lens, a, v, init, dh, dl)):
        check(x, want, bound, name)


def test_scan_some_gradients_and_outputs():
    lens, d = [20, 0, 300, 7], 33
    a, v, init, dh, dl = scan_inputs(1, lens, d, BF16, F32)
    want = scan_reference(lens, a, v, init, dh, dl)
    plan = ops.segment_plan(lens)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        leaves = [t.clone().requires_grad_(bool(k)) for t, k in zip((a, v, init), need)]
        h, last = ops.segment_scan(plan, *leaves, return_state=True)
        got = torch.autograd.grad((h, last), [t for t in leaves if t.requires_grad], (dh, dl))
        for x, (w, b) in zip(got, [want[2 + i] for i in range(3) if need[i]]):
            check(x, w, b, str(need))
    # only one of the outputs has a gradient; no initial states
    zero = torch.zeros_like(dh)
    A, V = a.clone().requires_grad_(), v.clone().requires_grad_()
    h, last = ops.segment_scan(plan, A, V, return_state=True)
    got = torch.autograd.grad(h, (A, V), dh, retain_graph=True)
    for x, (w, b) in zip(got, scan_reference(lens, a, v, None, dh, None)[2:4]):
        check(x, w, b, "h alone")
    got = torch.autograd.grad(last, (A, V), dl)
    for x, (w, b) in zip(got, scan_reference(lens, a, v, None, zero, dl)[2:4]):
        check(x, w, b, "last alone")


def test_scan_gradients_against_differences():
    a, v, init, _, _ = scan_inputs(2, [3, 0, 18, 1], 3, F64, F64)
    a, v, init = (t.requires_grad_() for t in (a, v, init))
    plan = ops.segment_plan([3, 0, 18, 1])
    assert torch.autograd.gradcheck(
        lambda *t: ops.segment_scan(plan, *t, return_state=True), (a, v, init))
    x, w, b = (rand(gen(3), *s, dtype=F64).requires_grad_() for s in ((4, 9), (9,), (9,)))
    assert torch.autograd.gradcheck(lambda *t: ops.layer_norm(*t), (x, w, b))


def test_scan_infinities_stay_in_their_segments():
    """A NaN or an infinity in a segment reaches none of its neighbours, in either
    direction, whether segments lie in one chunk or over many."""
    for lens in ([40, 3, 60], [700, 700, 300]):
        d, first, second = 20, lens[0], lens[0] + lens[1]
        a, v, init, dh, dl = scan_inputs(4, lens, d, F32, F32, low=0.9)

        def run(a, v, dh):
            A, V = a.clone().requires_grad_(), v.clone().requires_grad_()
            h, last = ops.segment_scan(lens, A, V, init, return_state=True)
            return [h.detach()] + list(torch.autograd.grad((h, last), (A, V), (dh, dl)))

        want = run(a, v, dh)
        for bad in (float("inf"), float("nan")):
            for which in range(3):
                x = [a.clone(), v.clone(), dh.clone()]
                x[which][first + 1, 3] = bad
                got = run(*x)
                for g, w in zip(got, want):
                    assert torch.equal(g[:first], w[:first])
                    assert torch.equal(g[second:], w[second:])
                    assert torch.equal(g[:, 4:], w[:, 4:])
        # gates whose product overflows, in front of a segment that starts from zeros
        b = a.clone()
        b[first:second] = 1e30
        z = v.clone()
        z[first:second] = 0.0
        zi = init.clone()
        zi[1] = 0.0
        h = ops.segment_scan(lens, b, z, zi)
        assert bool((h[first:second] == 0).all()) and torch.equal(h[second:], want[0][second:])


def test_scan_shapes_containers_and_plans():
    rng = np.random.default_rng(0)
    a, v = rng.random((7, 2, 3)), rng.standard_normal((7, 2, 3))
    lens = [4, 0, 3]
    got, last = ops.segment_scan(lens, a, v, return_state=True)
    assert isinstance(got, np.ndarray) and last.shape == (3, 2, 3)
    cur = 0.0
    for t in range(7):
        cur = a[t] * (0.0 if t == 4 else cur) + v[t]
        np.testing.assert_allclose(got[t], cur, rtol=1e-14, atol=1e-15)
    np.testing.assert_array_equal(last[[0, 2]], got[[3, 6]])
    assert not last[1].any()
    # the documented example
    ex = ops.segment_scan([2, 0, 3], np.full((5, 1), 0.5), np.ones((5, 1)))
    np.testing.assert_array_equal(ex[:, 0], [1.0, 1.5, 1.0, 1.5, 1.75])
    # lengths as a GPU tensor, a list, a plan; one value a row
    at, vt = torch.from_numpy(a[:, 0, 0]).cuda(), torch.from_numpy(v[:, 0, 0]).cuda()
    for seglen in (lens, torch.tensor(lens), torch.tensor(lens, device="cuda"),
                   ops.segment_plan(lens), ops.segment_plan(torch.tensor(lens, device="cuda"), 7)):
        assert torch.equal(ops.segment_scan(seglen, at, vt).cpu(), torch.from_numpy(got[:, 0, 0]))
    # no rows, no columns, no segments
    e = torch.zeros(0, 4, device="cuda")
    h, last = ops.segment_scan([0, 0], e, e, torch.ones(2, 4, device="cuda"), return_state=True)
    assert h.shape == (0, 4) and torch.equal(last, torch.ones(2, 4, device="cuda"))
    E, I = e.clone().requires_grad_(), torch.ones(2, 4, device="cuda", requires_grad=True)  # noqa: E741
    h, last = ops.segment_scan([0, 0], e, E, I, return_state=True)
    assert torch.equal(torch.autograd.grad(last.sum(), I)[0], torch.ones(2, 4, device="cuda"))
    assert ops.segment_scan([], e, e).shape == (0, 4)
    z = torch.zeros(5, 0, device="cuda")
    assert ops.segment_scan([5], z, z).shape == (5, 0)
    plan = ops.segment_plan([3, 2])
    with pytest.raises(DGLError, match="plan of 5 rows"):
        ops.segment_scan(plan, e, e)
    x = torch.zeros(5, 4, device="cuda")
    with pytest.raises(DGLError, match="initial states"):
        ops.segment_scan(plan, x, x, x)
    for bad in (torch.tensor([3, 3], device="cuda"), torch.tensor([6, -1], device="cuda")):
        with pytest.raises(DGLError, match="segment lengths"):
            ops.segment_scan(bad, x, x)


def test_scan_types_meet():
    """float64 beside anything computes in float64; 16-bit values keep float32
    gates; other gates become float32."""
    lens = [3, 2]
    a, v, init, _, _ = scan_inputs(6, lens, 8, F64, F64)
    assert ops.segment_scan(lens, a, v.float()).dtype == F64
    assert torch.equal(ops.segment_scan(lens, a.to(BF16), v.float()),
                       ops.segment_scan(lens, a.to(BF16).float(), v.float()))
    assert torch.equal(ops.segment_scan(lens, a.to(F16), v.to(BF16)),
                       ops.segment_scan(lens, a.to(F16).float(), v.to(BF16)))
    h, last = ops.segment_scan(lens, a.to(BF16), v.to(BF16), init, return_state=True)
    assert h.dtype == BF16 and last.dtype == F32
    G = a.to(F16).requires_grad_()
    (d,) = torch.autograd.grad(ops.segment_scan(lens, G, v.to(BF16)).sum(), G)
    assert d.dtype == F16


def test_scan_of_cpu_tensors():
    """Results and gradients come back to where the operands are."""
    lens = [40, 0, 90]
    args = scan_inputs(16, lens, 12, F32, F32)
    a, v, init, dh, dl = args

    def run(*t):
        a, v, init, dh, dl = t
        A, V, I = (x.detach().requires_grad_() for x in (a, v, init))  # noqa: E741
        h, last = ops.segment_scan(lens, A, V, I, return_state=True)
        return [h.detach(), last.detach()] + \
            list(torch.autograd.grad((h, last), (A, V, I), (dh, dl)))

    for got, want in zip(run(*(t.cpu() for t in args)), run(*args)):
        assert got.device.type == "cpu" and torch.equal(got, want.cpu())
    # gates on the GPU, values on the CPU: results where the values are
    A, V = a.detach().requires_grad_(), v.cpu().requires_grad_()
    h = ops.segment_scan(lens, A, V)
    da, dv = torch.autograd.grad(h, (A, V), dh.cpu())
    assert h.device.type == dv.device.type == "cpu" and da.device.type == "cuda"


def test_scan_strides_alignment_and_broadcasts():
    g = gen(7)
    lens = [50, 0, 83]
    wide = rand(g, 133, 70)
    gates = torch.rand(133, 70, generator=g, device="cuda")
    for cut in (slice(0, 64), slice(1, 34), slice(3, 70, 2)):
        a, v = gates[:, cut], wide[:, cut]
        assert torch.equal(ops.segment_scan(lens, a, v),
                           ops.segment_scan(lens, a.contiguous(), v.contiguous()))
    one = torch.rand(133, 1, generator=g, device="cuda")  # a gate a row, shared by its columns
    G = one.clone().requires_grad_()
    (d,) = torch.autograd.grad(ops.segment_scan(lens, G.expand(133, 70), wide).sum(), G)
    H = one.expand(133, 70).contiguous().requires_grad_()
    (e,) = torch.autograd.grad(ops.segment_scan(lens, H, wide).sum(), H)
    torch.testing.assert_close(d, e.sum(1, keepdim=True), rtol=1e-5, atol=1e-4)
    for dtype in (F16, F32):
        for off in (1, 3):
            flat = rand(g, off + 133 * 70, dtype=dtype)
            v = flat[off:].view(133, 70)
            assert torch.equal(ops.segment_scan(lens, gates.to(dtype), v),
                               ops.segment_scan(lens, gates.to(dtype), v.clone()))


@pytest.mark.parametrize("dtype,gdtype", SCAN_TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (16, 64), (37, 101), (4, 3, 7)])
def test_step(dtype, gdtype, shape):
    g = gen(8)
    a = torch.rand(*shape, generator=g, device="cuda", dtype=F64).to(gdtype)
    v, s = rand(g, *shape, dtype=dtype), rand(g, *shape, dtype=state(dtype))
    u = HALF_STEP[state(dtype)]
    want = a.double() * s.double() + v.double()
    bound = 2 * u * ((a.double() * s.double()).abs() + v.double().abs())
    h, new = ops.segment_scan_step(a, v, s)
    check(h, want, bound, "h")
    check(new, want, bound, "state")
    # one more row of the scan
    n = shape[0]
    h2, last = ops.segment_scan([1] * n, a, v, s, return_state=True)
    assert torch.equal(h, h2) and torch.equal(new, last)
    # in place
    mine = s.clone()
    h3, same = ops.segment_scan_step(a, v, mine, out=mine)
    assert same is mine and torch.equal(mine, new) and torch.equal(h3, h)


def test_step_refusals():
    a, v, s = (torch.rand(4, 6, device="cuda") for _ in range(3))
    for out in (torch.empty(4, 6), torch.empty(4, 6, device="cuda", dtype=F64),
                torch.empty(4, 5, device="cuda"), torch.empty(6, 4, device="cuda").t(),
                np.zeros((4, 6), np.float32)):
        with pytest.raises(DGLError, match="out must be"):
            ops.segment_scan_step(a, v, s, out=out)
    flat = torch.rand(48, device="cuda")
    for out, state_ in ((flat[6:30].view(4, 6), flat[:24].view(4, 6)), (a, s), (v, s)):
        with pytest.raises(DGLError, match="overlaps"):
            ops.segment_scan_step(a, v, state_, out=out)
    h, new = ops.segment_scan_step(np.ones((2, 2)), np.ones((2, 2)), np.ones((2, 2)))
    assert isinstance(new, np.ndarray) and (h == 2).all()
    e = torch.zeros(0, 3, device="cuda")
    assert ops.segment_scan_step(e, e, e)[0].shape == (0, 3)


# ---------------------------------------------------------------- how they are called


def bits(ts):
    return [t.clone() for t in ts]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_results_are_the_same_each_time():
    g = gen(9)
    x, w, b, dy = (rand(g, *s) for s in ((3000, 130), (130,), (130,), (3000, 130)))
    lens = [1000, 0, 2000]
    gates = torch.rand(3000, 130, generator=g, device="cuda")

    def run():
        X, W, B, A = (t.clone().requires_grad_() for t in (x, w, b, gates))
        y = ops.segment_scan(lens, A, ops.layer_norm(X, W, B))
        return torch.autograd.grad(y, (X, W, B, A), dy)

    first = bits(run())
    for _ in range(5):
        assert same(run(), first)


def test_scan_results_do_not_depend_on_timing():
    """Chains of hundreds of chunks beside other work on the GPU, which changes how far
    each chunk has to look back: the same bits."""
    g = gen(20)
    n, d = 120_000, 200
    a = 0.99 + 0.01 * torch.rand(n, d, generator=g, device="cuda")
    v, dh = rand(g, n, d), rand(g, n, d)
    plan = ops.segment_plan([n - 50_000, 50_000])

    def run():
        A, V = a.detach().requires_grad_(), v.detach().requires_grad_()
        h = ops.segment_scan(plan, A, V)
        return [h.detach()] + list(torch.autograd.grad(h, (A, V), dh))

    first = bits(run())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for i in range(12):
        with torch.cuda.stream(side):
            for _ in range(i):
                ops.layer_norm(v[: 10_000 * (i + 1)])
        assert same(run(), first)
    torch.cuda.synchronize()


def test_a_plan_dropped_while_another_stream_reads_it():
    g = gen(21)
    x = rand(g, 4000, 64)
    want = ops.segment_scan([1500, 2500], torch.sigmoid(x), x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    plan = ops.segment_plan([1500, 2500])
    with torch.cuda.stream(side):
        z = x
        for _ in range(50):
            z = z * 1.0
        got = ops.segment_scan(plan, torch.sigmoid(z), z)
    del plan
    junk = [torch.full((4000,), -1, dtype=torch.int32, device="cuda") for _ in range(8)]
    side.synchronize()
    assert torch.equal(got, want) and len(junk) == 8


def test_other_streams():
    """Each call runs on the current stream, behind what its inputs wait for there; a
    plan made on one stream serves another."""
    g = gen(10)
    x, w = rand(g, 2000, 200), rand(g, 200)
    lens = torch.tensor([700, 1300], device="cuda")
    plan = ops.segment_plan(lens)

    def run(x):
        X, W = x.clone().requires_grad_(), w.clone().requires_grad_()
        y = ops.segment_scan(plan, torch.sigmoid(X), ops.layer_norm(X, W))
        s = ops.segment_scan_step(X[:3].detach(), X[3:6].detach(), X[6:9].detach())
        return [y.detach()] + list(s) + list(torch.autograd.grad(y, (X, W), x))

    want = bits(run(x * 3))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        z = x
        for _ in range(20):  # work the inputs wait for
            z = z * 1.0
        got = run(z * 3)
    side.synchronize()
    assert same(got, want)


def test_threads():
    g = gen(11)
    xs = [rand(g, 900 + 50 * i, 96) for i in range(4)]

    def run(x):
        n = x.shape[0]
        X = x.clone().requires_grad_()
        y = ops.segment_scan([n // 3, n - n // 3], torch.sigmoid(X), ops.layer_norm(X))
        return [y.detach()] + list(torch.autograd.grad(y, X, x))

    want = [bits(run(x)) for x in xs]
    torch.cuda.synchronize()
    results = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            results[i] = [run(xs[i]) for _ in range(5)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for r, w in zip(results, want):
        assert all(same(one, w) for one in r)


def test_captured_into_a_graph():
    """Forward and backward in a HIP graph, replayed with new inputs and with eager
    work between; two graphs whose workspaces are their own."""
    g = gen(12)
    n, d = 1500, 72
    plan = ops.segment_plan([400, 0, 1100])
    w, b, dy = rand(g, d), rand(g, d), rand(g, n, d)
    static = rand(g, n, d)
    states = rand(g, 3, d)

    def run(x, w, b):
        X, W, B = (t.detach().requires_grad_() for t in (x, w, b))
        y, last = ops.segment_scan(plan, torch.sigmoid(X), ops.layer_norm(X, W, B), states,
                                   return_state=True)
        grads = torch.autograd.grad((y, last), (X, W, B), (dy, states))
        step = ops.segment_scan_step(x[:3], x[3:6], states)
        return [y.detach(), last.detach()] + list(grads) + list(step)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(static, w, b)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(static, w, b)
        graphs.append((graph, out))
    for seed in range(4):
        static.copy_(rand(gen(100 + seed), n, d))
        want = bits(run(static, w, b))
        for graph, out in graphs:
            for t in out:
                t.zero_()
        for graph, out in graphs:
            graph.replay()
            ops.layer_norm(static)  # eager work between
        torch.cuda.synchronize()
        for _, out in graphs:
            assert same(out, want)


def test_rows_beyond_32_bits():
    """More than 2**31 values a tensor."""
    n, d = 1_050_000, 2080
    x = torch.empty(n, d, dtype=BF16, device="cuda").normal_(generator=gen(13))
    assert x.numel() > 2 ** 31
    pick = torch.tensor([0, 1, n // 2, n - 2, n - 1], device="cuda")
    y = ops.layer_norm(x)
    assert torch.equal(y[pick], ops.layer_norm(x[pick]))
    a = torch.full_like(x, 0.5)
    lens = [n - 40, 40]
    h = ops.segment_scan(lens, a, x)
    tail = ops.segment_scan([40], a[-40:], x[-40:])
    assert torch.equal(h[-40:], tail)
    # 2^-30 of what lies 30 rows back is below half a step of bfloat16
    part = ops.segment_scan([60], a[n - 100:n - 40], x[n - 100:n - 40])
    torch.testing.assert_close(h[n - 60:n - 40].float(), part[-20:].float(), rtol=2.0 ** -7,
                               atol=2.0 ** -20)
    torch.testing.assert_close(h[:20].float(), ops.segment_scan([20], a[:20], x[:20]).float())


def test_second_derivative_is_refused():
    x = torch.randn(4, 6, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(ops.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    assert dgl.layer_norm is ops.layer_norm

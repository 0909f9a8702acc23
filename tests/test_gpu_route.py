"""Routing to experts on the GPU (topk_route, route_plan, dispatch_rows,
combine_rows) against plain float64, and a layer made of all the row operators.

Choices have to be equal; weights and gradients lie within bounds that count their
roundings (u: half a step of float32, float64 for float64 rows)."""

import numpy as np
import pytest
import torch

import mojodgl.ops as ops
from mojodgl import DGLError

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
HALF_STEP = {F32: 2.0 ** -24, F64: 2.0 ** -53, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -126, F64: 1e-300, BF16: 2.0 ** -126, F16: 2.0 ** -24}
INF = float("inf")


def state(dtype):
    return F64 if dtype == F64 else F32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=F64).to(dtype)


def within(got, want, bound, name):
    limit = bound * (1 + HALF_STEP[got.dtype]) + want.abs() * HALF_STEP[got.dtype] \
        + TINY[got.dtype]
    off = (got.double() - want).abs()
    assert got.shape == want.shape and bool((off <= limit).all()), \
        "{}: {}".format(name, (off - limit).max().item())


# ---------------------------------------------------------------- the choice


def choose(x, k, score, bias, groups, topk_groups, group_score, renormalize, scale, dw):
    """Choices, weights, gradient of one call in float64, row by row in numpy."""
    x = x.double().cpu().numpy()
    bias = None if bias is None else bias.double().cpu().numpy()
    dw = dw.double().cpu().numpy()
    n, e = x.shape
    ids, weights, grad = np.zeros((n, k), np.int64), np.zeros((n, k)), np.zeros((n, e))
    for r in range(n):
        row = x[r]
        masked = np.isneginf(row)
        if score == "sigmoid":
            with np.errstate(over="ignore"):
                s = 1 / (1 + np.exp(-row))
            ds = s * (1 - s)
        else:
            top = row.max()
            p = np.zeros(e) if masked.all() else np.exp(row - top)
            s = p / p.sum() if not masked.all() else p
        key = np.where(masked, -INF, row if bias is None else s + bias)
        allowed = np.ones(e, bool)
        if topk_groups < groups:
            size = e // groups
            marks = []
            for g in range(groups):
                best = np.sort(key[g * size:(g + 1) * size])[::-1]
                mark = best[0]
                if group_score == "top2" and size > 1 and best[1] > -INF:
                    mark = mark + best[1]
                marks.append(mark)
            kept = sorted(range(groups), key=lambda g: (-marks[g], g))[:topk_groups]
            allowed = np.isin(np.arange(e) // size, kept)
        order = sorted(np.nonzero(allowed)[0], key=lambda i: (-key[i], i))[:k]
        ids[r] = order
        if renormalize:
            live = row[order].max() > -INF
            z = row[order] - row[order].max() if live else np.full(k, -INF)
            # scores that underflow keep their ratio, exp(x) for both kinds of score
            c = s[order] if score == "sigmoid" and live and row[order].max() > -600 else np.exp(z)
            w = c / c.sum() if c.sum() else c
        else:
            w = s[order]
        weights[r] = w * scale
        d = dw[r] * scale
        inner = (d * w).sum()
        if score == "softmax" and not renormalize:
            grad[r] = -s * inner
            grad[r, order] += s[order] * d
        elif score == "softmax":
            grad[r, order] = w * (d - inner)
        else:
            grad[r, order] = w * (1 - s[order]) * (d - inner) if renormalize else ds[order] * d
    return (torch.from_numpy(t).cuda() for t in (ids, weights, grad))


CHOICES = [  # experts, k, groups, topk_groups
    (1, 1, 1, 1), (3, 3, 1, 1), (8, 2, 1, 1), (16, 15, 1, 1), (17, 4, 1, 1), (40, 16, 1, 1),
    (64, 6, 8, 3), (64, 8, 4, 2), (65, 1, 5, 2), (100, 10, 10, 4), (128, 8, 1, 1), (160, 6, 8, 3),
    (255, 3, 3, 1), (256, 8, 8, 4), (256, 20, 16, 8), (257, 8, 1, 1), (300, 12, 20, 5),
    (512, 31, 8, 4), (512, 8, 64, 7), (513, 32, 3, 2), (1000, 5, 8, 1), (1024, 32, 32, 9),
    (1025, 9, 1, 1), (2048, 8, 8, 4), (2047, 32, 1, 1)]


def route_case(x, k, groups, top, seed, **kw):
    g = gen(seed)
    n, e = x.shape
    st = state(x.dtype)
    args = dict(score="softmax", bias=None, group_score="max", renormalize=True, scale=1.0)
    args.update(kw)
    dw = rand(g, n, k, dtype=st)
    ids0, w0, dx0 = choose(x, k, groups=groups, topk_groups=top, dw=dw, **args)
    X = x.clone().requires_grad_()
    w, ids = ops.topk_route(X, k, num_groups=groups, topk_groups=top, **args)
    assert ids.dtype == torch.int64 and w.dtype == st and not ids.requires_grad
    assert torch.equal(ids, ids0), int((ids != ids0).sum())
    u = HALF_STEP[st]
    # a score: the argument's rounding (the difference to the row's largest logit, up
    # to `span`, once more by log2 e) and 8 for exp, sum and quotient, then E / 16 + 8
    # for the row's sum in order over a lane and pairwise over lanes
    finite = torch.where(x.double().isfinite(), x.double(), 0.0)
    # (beyond 1,000 exp is 0 or infinite in every type, and no rounding shows)
    span = 2 * finite.abs().amax(1, keepdim=True).clamp(max=1000.0)
    rel = u * (4 * span + 24 + e / 16)
    within(w.detach(), w0, rel * w0.abs(), "weights")
    w2, ids2 = ops.topk_route(x, k, num_groups=groups, topk_groups=top, **args)
    assert torch.equal(w2, w.detach()) and torch.equal(ids2, ids)
    (dx,) = torch.autograd.grad(w, X, dw)
    assert dx.dtype == x.dtype
    # products of weights and d = scale dw, the inner product over k terms
    d = (args["scale"] * dw.double()).abs()
    inner = (d * (w0 / args["scale"]).abs()).sum(1, keepdim=True)
    at = torch.zeros_like(dx0).scatter(1, ids0, d)
    s = torch.zeros_like(dx0).scatter(1, ids0, (w0 / args["scale"]).abs())
    if args["score"] == "softmax" and not args["renormalize"]:
        s = torch.softmax(torch.where(x.double() == -INF, -1e300, x.double()), 1)
    within(dx, dx0, (3 * rel + (k + 8) * u) * s * (at + inner), "gradient")
    return ids, w.detach()


@pytest.mark.parametrize("e,k,groups,top", CHOICES)
@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
def test_topk_route(e, k, groups, top, dtype):
    n = 37
    for i, (score, renorm, biased, gs) in enumerate([
            ("softmax", True, False, "max"), ("softmax", False, True, "top2"),
            ("sigmoid", True, True, "top2"), ("sigmoid", False, False, "top2"),
            ("sigmoid", False, True, "max"), ("softmax", False, False, "max")]):
        g = gen(100 * e + i)
        x = (1.5 * rand(g, n, e)).to(dtype)
        bias = 0.1 * rand(g, e, dtype=state(dtype)) if biased else None
        route_case(x, k, groups, top, i, score=score, renormalize=renorm, bias=bias,
                   group_score=gs, scale=(1.0, 2.5)[i % 2])


def test_equal_logits_go_to_the_lowest_index():
    x = torch.zeros(20, 96, device="cuda")
    x[:, 7] = -0.0
    for kw in (dict(), dict(bias=torch.zeros(96, device="cuda")), dict(score="sigmoid"),
               dict(score="sigmoid", bias=torch.full((96,), 0.5, device="cuda"))):
        _, ids = ops.topk_route(x, 5, **kw)
        assert torch.equal(ids, torch.arange(5, device="cuda").expand(20, 5))
        _, ids = ops.topk_route(x, 5, num_groups=6, topk_groups=2, group_score="top2", **kw)
        assert torch.equal(ids, torch.arange(5, device="cuda").expand(20, 5))
    g = gen(1)  # logits of few values: ties everywhere
    for dtype in (F32, BF16):
        x = torch.randint(-2, 3, (200, 130), generator=g, device="cuda").to(dtype)
        for bias in (None, 0.25 * torch.randint(0, 3, (130,), generator=g, device="cuda").float()):
            for groups, top in ((1, 1), (10, 3), (13, 5)):
                route_case(x, 9, groups, top, 3, bias=bias, group_score="top2", score="sigmoid")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_keys_that_differ_by_less_than_float32_shows(score):
    """Biases that bring the keys of a row's experts within 1e-9 of each other: the
    order is that of float64."""
    g = gen(2)
    n, e = 64, 48
    x = rand(g, 1, e).expand(n, e).contiguous()
    x = x + 1e-3 * rand(g, n, e)  # float32 logits, all different
    s = (torch.softmax if score == "softmax" else lambda t, _: torch.sigmoid(t))(x.double(), 1)
    bias = (1.0 - s[0]).float()  # row 0: keys of 1 but for float32's rounding
    for k, groups, top in ((6, 1, 1), (4, 8, 2)):
        route_case(x[:1].expand(8, e).contiguous(), k, groups, top, 5, score=score, bias=bias,
                   renormalize=False, group_score="top2")
        route_case(x, k, groups, top, 5, score=score, bias=bias, renormalize=False)
    # without a bias the marks of groups are sums of two logits
    y = torch.tensor([[1.0, 2.0 ** -24, 1.0 + 2.0 ** -23, -2.0 ** -23, 0.5, 0.5, 0.0, 0.0]],
                     device="cuda").expand(6, 8).contiguous()
    route_case(y, 2, 4, 1, 6, group_score="top2")


def test_masks():
    """-inf masks experts, whole groups, whole rows; the lowest finite values do not."""
    g = gen(3)
    n, e = 40, 64
    for dtype in (F32, BF16, F16, F64):
        for kw in (dict(), dict(score="sigmoid"), dict(renormalize=False),
                   dict(score="sigmoid", renormalize=False),
                   dict(score="sigmoid", bias=0.1 * rand(g, e, dtype=state(dtype))),
                   dict(bias=0.1 * rand(g, e, dtype=state(dtype)), renormalize=False)):
            x = rand(g, n, e, dtype=dtype)
            x[0] = -INF                 # nothing left
            x[1, 1:] = -INF             # one expert, fewer than k
            x[2, :63] = -INF
            x[3, ::2] = -INF
            x[4, 8:] = -INF             # one group of eight
            x[5] = torch.finfo(dtype).min
            x[6, :60] = torch.finfo(dtype).min
            x[7:] = torch.where(rand(g, n - 7, e) > 0.5, x[7:], -INF)
            for groups, top, gs in ((1, 1, "max"), (8, 3, "max"), (8, 2, "top2"), (4, 3, "top2")):
                ids, w = route_case(x, 5, groups, top, 7, group_score=gs, **kw)
                assert bool((w[0] == 0).all()) and bool(w.isfinite().all())
                assert bool((w[1] == 0)[1:].all() if groups == 1 else True)


def test_sums_of_the_lowest_values_stay_above_masked_groups():
    low = torch.finfo(F32).min
    x = torch.tensor([[-INF, -INF, low, low, low, low / 2, -INF, -INF],
                      [-INF, -INF, low, -INF, low, low, 1.0, -INF]], device="cuda")
    for top in (1, 2, 3):
        route_case(x, 2, 4, top, 12, group_score="top2")


def test_rows_with_nan_or_inf():
    """Their weights show it, their ids stay in range, other rows are as they were."""
    g = gen(4)
    x = rand(g, 32, 100)
    for kw in (dict(), dict(renormalize=False), dict(bias=rand(g, 100)),
               dict(num_groups=10, topk_groups=3, group_score="top2", bias=rand(g, 100))):
        w0, ids0 = ops.topk_route(x, 6, **kw)
        y = x.clone()
        y[3, 50], y[9, 0], y[20] = float("nan"), INF, float("nan")
        w, ids = ops.topk_route(y, 6, **kw)
        assert bool(((ids >= 0) & (ids < 100)).all())
        assert all(len(set(r)) == 6 for r in ids.tolist())
        rest = [i for i in range(32) if i not in (3, 9, 20)]
        assert torch.equal(w[rest], w0[rest]) and torch.equal(ids[rest], ids0[rest])
        assert bool(w[20].isnan().all()) and bool(w[9].isnan().any())


def test_scores_that_underflow():
    """Renormalised weights of scores far below the smallest float32."""
    x = torch.tensor([[-200.0, -201.0, -250.0, -203.0], [-88.0, -89.0, -87.5, -95.0],
                      [200.0, -200.0, 100.0, 0.0], [-3e38, -3e38, -3.1e38, -3.2e38]],
                     device="cuda")
    route_case(x, 3, 1, 1, 8, score="sigmoid")
    route_case(x, 3, 1, 1, 8, score="softmax")
    route_case(x.double(), 3, 1, 1, 8, score="sigmoid")


def test_route_gradients_against_differences():
    g = gen(5)
    x = (3 * rand(g, 5, 12, dtype=F64)).requires_grad_()
    bias = 0.01 * rand(g, 12, dtype=F64)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            assert torch.autograd.gradcheck(
                lambda t: ops.topk_route(t, 3, score=score, renormalize=renorm, bias=bias,
                                         num_groups=3, topk_groups=2, scale=1.5)[0], x)


def test_route_shapes_and_containers():
    w, ids = ops.topk_route(np.random.default_rng(0).standard_normal((4, 9)), 2)
    assert isinstance(w, np.ndarray) and w.dtype == np.float64 and ids.dtype == np.int64
    np.testing.assert_allclose(w.sum(1), 1.0, rtol=1e-14)
    x = torch.randn(4, 9, requires_grad=True)  # on the CPU
    w, ids = ops.topk_route(x, 2)
    assert w.device.type == "cpu" and ids.device.type == "cpu"
    assert torch.autograd.grad(w[:, 0].sum(), x)[0].device.type == "cpu"
    e = torch.zeros(0, 9, device="cuda", requires_grad=True)
    w, ids = ops.topk_route(e, 2)
    assert w.shape == ids.shape == (0, 2)
    assert torch.autograd.grad(w.sum(), e)[0].shape == (0, 9)
    g = gen(6)
    wide = rand(g, 50, 71, dtype=BF16)
    for cut in (wide[:, 1:], wide[:, 3:67], wide[::3], wide.t()):
        for a, b in zip(ops.topk_route(cut, 4), ops.topk_route(cut.contiguous(), 4)):
            assert torch.equal(a, b)
    flat = rand(g, 1 + 20 * 64, dtype=F16)
    for a, b in zip(ops.topk_route(flat[1:].view(20, 64), 4),
                    ops.topk_route(flat[1:].view(20, 64).clone(), 4)):
        assert torch.equal(a, b)
    x = torch.randn(4, 9, device="cuda")
    for kw, text in ((dict(k=0), "experts a row"), (dict(k=10), "experts a row"),
                     (dict(k=33), "experts a row"), (dict(k=2, num_groups=2), "divide"),
                     (dict(k=2, num_groups=3, topk_groups=4), "of 3 groups"),
                     (dict(k=4, num_groups=3, topk_groups=1), "its groups")):
        with pytest.raises(DGLError, match=text):
            ops.topk_route(x, **kw)
    with pytest.raises(DGLError, match="2048 experts"):
        ops.topk_route(torch.zeros(2, 2049, device="cuda"), 1)


# ---------------------------------------------------------------- the way there and back


def plan_reference(ids, experts):
    flat = ids.cpu().numpy().reshape(-1)
    bins = np.where((flat >= 0) & (flat < experts), flat, experts)
    order = np.argsort(bins, kind="stable")
    slot = np.empty_like(order)
    slot[order] = np.arange(order.size)
    return (np.bincount(bins, minlength=experts + 1)[:experts], order,
            np.where(bins < experts, slot, ~slot).reshape(ids.shape))


@pytest.mark.parametrize("n,k,experts", [
    (1, 1, 1), (5, 1, 3), (64, 1, 64), (63, 2, 7), (256, 8, 256), (257, 8, 2048), (1024, 2, 5),
    (1025, 2, 5), (700, 3, 2047), (4000, 8, 100), (5000, 1, 1), (33000, 4, 60)])
def test_route_plan(n, k, experts):
    g = gen(n + experts)
    for low, high in ((0, experts), (-2, experts + 3), (experts // 2, experts // 2 + 1), (-9, 0)):
        ids = torch.randint(low, high, (n, k), generator=g, device="cuda")
        plan = ops.route_plan(ids, experts)
        seglen, order, slot = plan_reference(ids, experts)
        np.testing.assert_array_equal(plan.seglen.cpu().numpy(), seglen)
        np.testing.assert_array_equal(plan.order.cpu().numpy(), order)
        np.testing.assert_array_equal(plan.slot.cpu().numpy(), slot)
        assert plan.seglen.dtype == torch.int64


def test_route_plan_takes_ids_as_they_come():
    ids = np.array([[2, 0], [1, 1], [5, -1]])
    want = ops.route_plan(torch.from_numpy(ids).cuda(), 3)
    for other in (ids, ids.astype(np.int32), ids.tolist(), torch.from_numpy(ids),
                  torch.from_numpy(ids).cuda().int(), torch.from_numpy(ids).cuda().t()
                  .contiguous().t(), torch.from_numpy(ids).cuda().float()):
        plan = ops.route_plan(other, 3)
        for a, b in zip((plan.seglen, plan.order, plan.slot),
                        (want.seglen, want.order, want.slot)):
            assert torch.equal(a, b)
    assert ops.route_plan(ids[:, 0], 3).slot.shape == (3, 1)
    empty = ops.route_plan(np.zeros((0, 4), np.int64), 3)
    assert not empty.seglen.any() and empty.order.shape == (0,)
    with pytest.raises(DGLError, match="2048 experts"):
        ops.route_plan(ids, 2049)
    with pytest.raises(DGLError, match="whole numbers"):
        ops.route_plan(torch.tensor([0.5], device="cuda"), 3)


@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("d", [1, 3, 4, 7, 8, 9, 31, 64, 100, 128, 130, 511, 512, 600, 2048, 2051])
def test_dispatch_and_combine(dtype, d):
    for n, k, experts in ((1, 1, 2), (23, 2, 5), (70, 5, 9), (40, 9, 20)):
        g = gen(d + n)
        ids = torch.randint(-1, experts + 1, (n, k), generator=g, device="cuda")
        x, ys, dxs, dy = (rand(g, m, d, dtype=dtype) for m in (n, n * k, n * k, n))
        w = rand(g, n, k, dtype=state(dtype))
        plan = ops.route_plan(ids, experts)
        X, Y, W = (t.clone().requires_grad_() for t in (x, ys, w))
        xs, y = ops.dispatch_rows(X, plan), ops.combine_rows(Y, W, plan)
        assert xs.dtype == y.dtype == dtype
        dx, dys, dw = torch.autograd.grad((xs, y), (X, Y, W), (dxs, dy))
        assert dw.dtype == state(dtype) and dx.dtype == dys.dtype == dtype
        slot = plan.slot.long()
        ok = slot >= 0
        place = torch.where(ok, slot, ~slot)
        want = torch.zeros_like(ys)
        want[place[ok]] = x.unsqueeze(1).expand(n, k, d)[ok]
        assert torch.equal(xs.detach(), want)
        u = HALF_STEP[state(dtype)]
        live = ok.double().unsqueeze(2)
        terms = w.double().unsqueeze(2) * ys.double()[place] * live
        within(y.detach(), terms.sum(1), k * u * terms.abs().sum(1), "combine")
        back = dxs.double()[place] * live
        within(dx, back.sum(1), k * u * back.abs().sum(1), "dx")
        prod = w.double().unsqueeze(2) * dy.double().unsqueeze(1)
        want = torch.zeros(n * k, d, dtype=F64, device="cuda")
        want[place.reshape(-1)] = (prod * live).reshape(-1, d)
        within(dys, want, 2 * u * want.abs(), "dys")
        dots = ys.double()[place] * dy.double().unsqueeze(1) * live
        # in order over d / 64 columns a lane (V of them), pairwise over lanes
        within(dw, dots.sum(2), u * (d / 16 + 40) * dots.abs().sum(2), "dw")
        assert torch.equal(ops.combine_rows(ys, w, plan), y.detach())


def test_entries_of_no_expert_are_not_read():
    """Rows behind the last expert's may hold anything."""
    ids = torch.tensor([[0, -1], [7, 1]], device="cuda")
    plan = ops.route_plan(ids, 2)
    y = torch.ones(4, 40, device="cuda")
    y[2:] = float("nan")
    w = torch.tensor([[2.0, float("nan")], [float("inf"), 3.0]], device="cuda")
    Y, W = y.requires_grad_(), w.requires_grad_()
    out = ops.combine_rows(Y, W, plan)
    assert torch.equal(out[0], torch.full((40,), 2.0, device="cuda"))
    assert torch.equal(out[1], torch.full((40,), 3.0, device="cuda"))
    dys, dw = torch.autograd.grad(out.sum(), (Y, W))
    assert torch.equal(dw, torch.tensor([[40.0, 0.0], [0.0, 40.0]], device="cuda"))
    assert torch.equal(dys[:, 0], torch.tensor([2.0, 3.0, 0.0, 0.0], device="cuda"))


def test_moves_shapes_containers_and_refusals():
    rng = np.random.default_rng(1)
    ids, x, w = rng.integers(0, 3, (6, 2)), rng.standard_normal((6, 2, 5)), rng.random((6, 2))
    plan = ops.route_plan(ids, 3)
    xs = ops.dispatch_rows(x, plan)
    assert isinstance(xs, np.ndarray) and xs.shape == (12, 2, 5)
    np.testing.assert_array_equal(xs, x[plan.order.cpu().numpy() // 2])
    np.testing.assert_allclose(ops.combine_rows(xs, w, plan), x * w.sum(1)[:, None, None],
                               rtol=1e-14)
    one = ops.route_plan(ids[:, 0], 3)
    np.testing.assert_allclose(ops.combine_rows(ops.dispatch_rows(x, one), w[:, 0], one),
                               x * w[:, 0][:, None, None], rtol=1e-14)
    assert ops.dispatch_rows(x.astype(np.float16), plan).dtype == np.float16
    t = torch.from_numpy(x).requires_grad_()
    assert ops.dispatch_rows(t, plan).device.type == "cpu"
    assert torch.equal(torch.autograd.grad(ops.dispatch_rows(t, plan).sum(), t)[0],
                       torch.full_like(t, 2.0))
    with pytest.raises(DGLError, match="of 6 rows"):
        ops.dispatch_rows(x[:5], plan)
    with pytest.raises(DGLError, match="12 entries"):
        ops.combine_rows(xs[:11], w, plan)
    with pytest.raises(DGLError, match="weights must have shape"):
        ops.combine_rows(xs, w[:, :1], plan)
    with pytest.raises(DGLError, match="made by route_plan"):
        ops.dispatch_rows(x, [1, 2])
    with pytest.raises(DGLError, match="made by route_plan"):
        ops.combine_rows(x, w, None)
    for shape in ((6, 0), (6, 2, 0)):
        z = torch.zeros(shape, device="cuda", requires_grad=True)
        zs = ops.dispatch_rows(z, plan)
        W = torch.ones(6, 2, device="cuda", requires_grad=True)
        y = ops.combine_rows(zs, W, plan)
        assert y.shape == shape
        dz, dw = torch.autograd.grad(y.sum(), (z, W))
        assert dz.shape == shape and not dw.any()
    empty = ops.route_plan(np.zeros((0, 2), np.int64), 3)
    assert ops.dispatch_rows(np.zeros((0, 5)), empty).shape == (0, 5)
    assert ops.combine_rows(np.zeros((0, 5)), np.zeros((0, 2)), empty).shape == (0, 5)
    none = ops.route_plan(np.zeros((6, 0), np.int64), 3)  # no choices: sums of nothing
    assert not ops.combine_rows(np.zeros((0, 5)), np.zeros((6, 0)), none).any()
    g = gen(7)
    flat = rand(g, 3 + 6 * 10 + 12 * 10, dtype=BF16)
    a, b = flat[1:61].view(6, 10), flat[63:].view(12, 10)
    assert torch.equal(ops.dispatch_rows(a, plan), ops.dispatch_rows(a.clone(), plan))
    assert torch.equal(ops.combine_rows(b, w, plan), ops.combine_rows(b.clone(), w, plan))


def test_moves_beyond_32_bits():
    """More than 2**31 values in the experts' rows."""
    n, k, d = 131_100, 8, 2056
    assert n * k * d > 2 ** 31
    g = gen(8)
    ids = torch.randint(0, 64, (n, k), generator=g, device="cuda")
    plan = ops.route_plan(ids, 64)
    x = torch.empty(n, d, dtype=BF16, device="cuda").normal_(generator=g)
    xs = ops.dispatch_rows(x, plan)
    pick = torch.randint(0, n * k, (4000,), generator=g, device="cuda")
    pick[:2] = torch.tensor([0, n * k - 1], device="cuda")
    assert torch.equal(xs[pick], x[plan.order[pick].long() // k])
    X = xs.requires_grad_()
    W = torch.full((n, k), 0.125, device="cuda", requires_grad=True)
    y = ops.combine_rows(X, W, plan)
    assert torch.equal(y.detach(), x)  # eight equal eighths
    dys, dw = torch.autograd.grad(y, (X, W), x)
    assert torch.equal(dys[pick], (x.float() * 0.125).to(BF16)[plan.order[pick].long() // k])
    rows = torch.tensor([0, 5, n - 1], device="cuda")
    want = x[rows].double().square().sum(1, keepdim=True).expand(3, k)
    torch.testing.assert_close(dw[rows].double(), want, rtol=2.0 ** -15, atol=0.0)


# ---------------------------------------------------------------- together


def layer(x, p, plan, k, experts):
    """One layer over packed rows: mixing along each sequence, then experts."""
    t = ops.layer_norm(x, p["w1"], p["b1"])
    h, last = ops.segment_scan(plan, torch.sigmoid(t @ p["gate"]), t @ p["value"], p["init"],
                               return_state=True)
    x = x + h
    t = ops.layer_norm(x, p["w2"], p["b2"])
    weights, ids = ops.topk_route(t @ p["router"], k, score="sigmoid", bias=p["balance"],
                                  num_groups=2, topk_groups=1, scale=1.5)
    route = ops.route_plan(ids, experts)
    y = ops.segment_mm(ops.dispatch_rows(t, route), p["experts"], route.seglen)
    return x + ops.combine_rows(y, weights, route), last, ids


def plain_layer(x, p, lens, ids):
    def norm(v, w, b):
        c = v - v.mean(1, keepdim=True)
        return c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * w + b

    t = norm(x, p["w1"], p["b1"])
    a, v = torch.sigmoid(t @ p["gate"]), t @ p["value"]
    rows, last, at = [], [], 0
    for s, m in enumerate(lens):
        cur = p["init"][s]
        for r in range(at, at + m):
            cur = a[r] * cur + v[r]
            rows.append(cur)
        last.append(cur)
        at += m
    x = x + torch.stack(rows)
    t = norm(x, p["w2"], p["b2"])
    s = torch.sigmoid(t @ p["router"]).gather(1, ids)
    weights = 1.5 * s / s.sum(1, keepdim=True)
    y = torch.stack([torch.stack([t[r] @ p["experts"][e] for e in ids[r].tolist()])
                     for r in range(len(ids))])
    return x + (weights.unsqueeze(2) * y).sum(1), torch.stack(last)


@pytest.mark.parametrize("dtype,tol", [(F64, 1e-10), (F32, 2e-4)])
def test_a_layer_of_them(dtype, tol):
    """Norm, scan, norm, routing, the experts' products and back: results and every
    parameter's gradient against torch's autograd in float64. (float32: the products
    of the test's own torch calls round too; 2e-4 is some hundred roundings of sums
    of 40 terms through eight stages.)"""
    g = gen(9)
    lens, d, experts, k = [30, 0, 25, 1], 40, 6, 2
    n = sum(lens)
    shapes = dict(w1=(d,), b1=(d,), w2=(d,), b2=(d,), gate=(d, d), value=(d, d),
                  init=(len(lens), d), router=(d, experts), experts=(experts, d, d))
    p = {name: rand(g, *s, dtype=dtype) * (d ** -0.5 if len(s) > 1 else 1.0)
         for name, s in shapes.items()}
    x, dy, dl = rand(g, n, d, dtype=dtype), rand(g, n, d, dtype=dtype), rand(g, 4, d, dtype=dtype)
    balance = 0.1 * rand(g, experts, dtype=dtype)
    leaves = [x] + list(p.values())

    def grads(fn, leaves):
        leaves = [t.detach().clone().requires_grad_() for t in leaves]
        y, last, *rest = fn(leaves[0], dict(zip(p, leaves[1:]), balance=balance))
        w = [t.to(y.dtype) for t in (dy, dl)]
        return [y.detach(), last.detach()] + list(torch.autograd.grad((y, last), leaves, w)), rest

    plan = ops.segment_plan(lens)
    got, (ids,) = grads(lambda x, p: layer(x, p, plan, k, experts), leaves)
    want, _ = grads(lambda x, p: plain_layer(x, p, lens, ids), [t.double() for t in leaves])
    for name, a, b in zip(["y", "last", "x"] + list(p), got, want):
        scale = b.abs().max()
        assert float((a.double() - b).abs().max()) <= tol * float(scale), name


def test_routing_captured_into_a_graph():
    """Choice, plan, ways and gradients in a HIP graph, replayed with other logits (and
    other numbers of rows for each expert), with eager work between; a second graph's
    workspaces are its own. Small and large plans."""
    for n, e, k in ((200, 16, 2), (3000, 64, 4)):
        g = gen(10)
        logits, x, dy = rand(g, n, e), rand(g, n, 72), rand(g, n, 72)
        bias = 0.1 * rand(g, e)

        def run():
            L, X = logits.detach().requires_grad_(), x.detach().requires_grad_()
            w, ids = ops.topk_route(L, k, score="sigmoid", bias=bias, num_groups=4,
                                    topk_groups=2, group_score="top2")
            plan = ops.route_plan(ids, e)
            y = ops.combine_rows(ops.dispatch_rows(X, plan), w, plan)
            return [ids, plan.seglen, plan.order, y.detach()] + \
                list(torch.autograd.grad(y, (L, X), dy))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = run()
            graphs.append((graph, out))
        for seed in range(4):
            logits.copy_(rand(gen(50 + seed), n, e))
            want = [t.clone() for t in run()]
            for _, out in graphs:
                for t in out:
                    t.zero_()
            for graph, out in graphs:
                graph.replay()
                ops.topk_route(logits, k)
            torch.cuda.synchronize()
            for _, out in graphs:
                assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_routing_on_another_stream_and_repeated():
    g = gen(11)
    logits, x = rand(g, 5000, 100), rand(g, 5000, 64, dtype=BF16)

    def run(logits, x):
        L, X = logits.detach().requires_grad_(), x.detach().requires_grad_()
        w, ids = ops.topk_route(L, 4)
        plan = ops.route_plan(ids, 100)
        y = ops.combine_rows(ops.dispatch_rows(X, plan), w, plan)
        return [y.detach(), ids] + list(torch.autograd.grad(y, (L, X), x))

    want = [t.clone() for t in run(logits * 2, x)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        z = logits
        for _ in range(20):
            z = z * 1.0
        for _ in range(3):
            got = run(z * 2, x)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))

"""Groups of experts ranked by the sum of their best two scores (topk_route with
group_score='top2'), without a bias as with one of zeros, against plain float64."""

import numpy as np
import pytest
import torch

import mojodgl.ops as ops

pytestmark = pytest.mark.gpu

F32, F64, BF16, F16 = torch.float32, torch.float64, torch.bfloat16, torch.float16
INF = float("inf")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=F64).to(dtype)


def scores(x, score):
    """float64 scores of numpy rows; 0 where a logit is -inf."""
    with np.errstate(over="ignore"):
        if score == "sigmoid":
            return 1 / (1 + np.exp(-x))
    top = x.max(1, keepdims=True)
    p = np.exp(x - np.where(np.isneginf(top), 0.0, top))
    total = p.sum(1, keepdims=True)
    return p / np.where(total > 0, total, 1.0)


def chosen(x, k, score, groups, top, bias=None, group_score="top2"):
    """The ids: experts by their logits, or by score + bias; groups by their best two
    scores (+ bias) together, a masked expert adding nothing."""
    x = x.double().cpu().numpy()
    n, e = x.shape
    masked = np.isneginf(x)
    rank = scores(x, score) + (0.0 if bias is None else bias.double().cpu().numpy())
    rank = np.where(masked, -INF, rank)
    key = x if bias is None else rank
    if group_score == "max":
        rank = key
    best = -np.sort(-rank.reshape(n, groups, e // groups), axis=2)
    mark = best[..., 0].copy()
    if group_score == "top2" and e > groups:
        mark += np.where(best[..., 1] > -INF, best[..., 1], 0.0)
    kept = np.argsort(-mark, axis=1, kind="stable")[:, :top]
    out = np.ones((n, groups), bool)
    np.put_along_axis(out, kept, False, axis=1)
    out = np.repeat(out, e // groups, axis=1)
    order = np.argsort(-key, axis=1, kind="stable")
    back = np.argsort(np.take_along_axis(out, order, 1), axis=1, kind="stable")
    ids = np.take_along_axis(order, back, 1)[:, :k]
    return torch.from_numpy(ids).cuda()


def check(x, k, score, groups, top, **kw):
    want = chosen(x, k, score, groups, top, **kw)
    for renormalize in (True, False):
        w, ids = ops.topk_route(x, k, score=score, num_groups=groups, topk_groups=top,
                                renormalize=renormalize,
                                **{"group_score": "top2", **kw})
        assert torch.equal(ids, want), int((ids != want).any(1).sum())
    # the last call's weights are the scores: half steps of float32 (float64), from
    # the argument, exp, the row's sum and the quotient
    x = x.double()
    s = torch.from_numpy(scores(x.cpu().numpy(), score)).cuda().gather(1, want)
    span = 2 * torch.where(x.isfinite(), x, 0.0).abs().amax(1, keepdim=True).clamp(max=1000.0)
    u = 2.0 ** (-53 if w.dtype == F64 else -24)
    assert bool(((w.double() - s).abs() <= u * (4 * span + 32 + x.shape[1] / 16) * s
                 + 2.0 ** -126).all())


GROUPS = [  # experts, k, groups, kept
    (64, 6, 8, 3), (64, 8, 4, 2), (65, 1, 5, 2), (100, 10, 10, 4), (160, 6, 8, 3), (12, 2, 12, 5),
    (255, 3, 3, 1), (256, 8, 8, 4), (256, 20, 16, 8), (300, 12, 20, 5), (512, 31, 8, 4),
    (512, 8, 64, 7), (513, 32, 3, 2), (1000, 5, 8, 1), (1024, 32, 32, 9), (2048, 8, 8, 4)]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [F32, F64, BF16, F16])
@pytest.mark.parametrize("e,k,groups,top", GROUPS)
def test_best_two_scores(e, k, groups, top, dtype, score):
    g = gen(e + k)
    n = 203
    for scale, shift in ((1.5, 0.0), (0.3, 0.0), (4.0, 2.0), (1.0, -9.0)):
        x = (scale * rand(g, n, e) + shift).to(dtype)
        check(x, k, score, groups, top)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_no_bias_chooses_as_a_bias_of_zeros(score):
    g = gen(1)
    for e, k, groups, top in ((256, 8, 8, 4), (96, 4, 6, 2), (1024, 8, 16, 5)):
        for dtype in (F32, F64, BF16):
            x = (1.5 * rand(g, 3000, e)).to(dtype)
            zero = torch.zeros(e, device="cuda", dtype=F64 if dtype == F64 else F32)
            got, want = (ops.topk_route(x, k, score=score, bias=b, num_groups=groups,
                                        topk_groups=top, group_score="top2")[1]
                         for b in (None, zero))
            assert torch.equal(got, want), int((got != want).any(1).sum())


def test_a_constant_added_to_a_row_changes_no_softmax_choice():
    g = gen(2)
    x = torch.randint(-3000, 3000, (2000, 64), generator=g, device="cuda").float() / 1024
    x[:, ::3] = -INF
    want = ops.topk_route(x, 5, num_groups=8, topk_groups=3, group_score="top2")[1]
    for shift in (-5.0, 8.0, -100.0):  # the sums are exact
        got = ops.topk_route(x + shift, 5, num_groups=8, topk_groups=3, group_score="top2")[1]
        assert torch.equal(got, want)
    # one expert of 1.0 against two of 0.8 and 0.7: e^1.0 < e^0.8 + e^0.7
    y = torch.tensor([[1.0, -INF, 0.8, 0.7]], device="cuda")
    for shift in (0.0, -5.0, 5.0, -90.0):
        for k in (1, 2):
            ids = ops.topk_route(y + shift, k, num_groups=2, topk_groups=1,
                                 group_score="top2")[1]
            assert ids.tolist() == [[2, 3][:k]]


def test_masks_and_the_lowest_values():
    g = gen(3)
    n, e = 60, 64
    for dtype in (F32, BF16, F16, F64):
        low = torch.finfo(dtype).min
        x = rand(g, n, e, dtype=dtype)
        x[0] = -INF
        x[1, 1:] = -INF
        x[2, :63] = -INF
        x[3, ::2] = -INF
        x[4, 8:] = -INF
        x[5] = low
        x[6, :60] = low
        x[7, :60] = -INF
        x[7, 60:] = low
        x[8] = -INF
        x[8, 40:43] = low
        x[8, 3] = low / 2
        x[9:30] = torch.where(rand(g, 21, e) > 0.5, x[9:30], -INF)
        x[30:] = torch.where(rand(g, 30, e) > 1.2, x[30:], -INF)
        for score in ("softmax", "sigmoid"):
            for groups, top in ((8, 2), (4, 3), (16, 5)):
                for k in (1, 4, 7):
                    check(x, k, score, groups, top)


@pytest.mark.parametrize("centre", [-30.0, -60.0, -86.0, -95.0, -200.0, 12.0])
def test_scores_far_from_one_half(centre):
    """Sigmoids that are tiny, below float32's smallest, or next to 1: the groups' order
    is that of float64."""
    g = gen(4)
    check(centre + rand(g, 500, 96), 4, "sigmoid", 12, 5)
    check((centre + rand(g, 500, 96)).to(BF16), 4, "sigmoid", 12, 5)


def test_sums_that_differ_by_less_than_float32_shows():
    """Two groups whose best two scores have almost the same sum."""
    g = gen(5)
    n = 4000
    for score in ("softmax", "sigmoid"):
        x = rand(g, n, 6, dtype=F64)
        x[:, 4:] = -9.0
        f = torch.exp if score == "softmax" else torch.sigmoid
        x[:, 1] = x[:, 0] - 0.3  # the second group: the same sum from other terms
        x[:, 2] = x[:, 0] - 0.1
        rest = f(x[:, 0].float().double()) + f(x[:, 1].float().double()) \
            - f(x[:, 2].float().double())
        x[:, 3] = rest.log() if score == "softmax" else torch.logit(rest)
        x = x.float()
        check(x, 2, score, 3, 1)
        check(x[:, [2, 3, 0, 1, 4, 5]].contiguous(), 2, score, 3, 1)


def test_groups_of_one_expert_and_groups_by_max_keep_the_logits_order():
    g = gen(6)
    x = rand(g, 400, 24)
    for score in ("softmax", "sigmoid"):
        check(x, 3, score, 24, 7)
        check(x, 3, score, 8, 2, group_score="max")
        check(x + 60.0, 3, "softmax", 24, 7)


def test_rows_with_nan_or_inf():
    """Ids stay in range and apart, other rows are as they were; an infinite logit's
    group comes first by softmax."""
    g = gen(7)
    for dtype in (F32, F64, BF16):
        for score in ("softmax", "sigmoid"):
            x = rand(g, 40, 96, dtype=dtype)
            how = dict(score=score, num_groups=12, topk_groups=3, group_score="top2")
            w0, ids0 = ops.topk_route(x, 5, **how)
            y = x.clone()
            y[3, 50], y[9, 41], y[20], y[21, 8:16] = float("nan"), INF, float("nan"), INF
            w, ids = ops.topk_route(y, 5, **how)
            assert bool(((ids >= 0) & (ids < 96)).all())
            assert all(len(set(r)) == 5 for r in ids.tolist())
            rest = [i for i in range(40) if i not in (3, 9, 20, 21)]
            assert torch.equal(w[rest], w0[rest]) and torch.equal(ids[rest], ids0[rest])
            assert ids[21].tolist() == [8, 9, 10, 11, 12]
            if score == "softmax":
                assert ids[9, 0] == 41
            else:  # a score of 1, and the group's second
                assert torch.equal(ids[9:10], chosen(y[9:10], 5, score, 12, 3))

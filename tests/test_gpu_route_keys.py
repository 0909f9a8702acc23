"""Experts whose keys (score + bias) nearly meet: topk_route's order is that of
float64, wherever the scores lie and whichever experts have the larger errors."""

import numpy as np
import pytest
import torch

import mojodgl.ops as ops

pytestmark = pytest.mark.gpu

F32, F64 = torch.float32, torch.float64


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=F64)


def uniform(g, low, high, *shape):
    return low + (high - low) * torch.rand(*shape, generator=g, device="cuda", dtype=F64)


def softmax(x):
    """In numpy: torch's own of float64 rows of more than 1,024 is off by 1e-6."""
    p = np.exp(x - x.max(1, keepdims=True))
    return torch.from_numpy(p / p.sum(1, keepdims=True)).cuda()


def check(x, bias, k, score, **kw):
    s = torch.sigmoid(x.double()) if score == "sigmoid" else softmax(x.double().cpu().numpy())
    key = s + bias.double()
    want = np.argsort(-key.cpu().numpy(), axis=1, kind="stable")[:, :k]
    ids = ops.topk_route(x, k, score=score, bias=bias, **kw)[1].cpu().numpy()
    assert (ids == want).all(), "{} of {} rows".format(int((ids != want).any(1).sum()), len(x))


@pytest.mark.parametrize("centre", [-1.0, -10.0, -20.0, -30.0, -45.0, -60.0, -75.0])
def test_sigmoids_far_below_zero(centre):
    """Two keys made equal by biases of the scores' own size but for the logits'
    rounding, which is of the size of the float scores' errors."""
    g = gen(int(-centre))
    n = 6000
    for _ in range(6):
        x = uniform(g, centre - 0.5, centre + 0.5, n, 1)
        gap = torch.sigmoid(torch.tensor(centre - 0.7, dtype=F64, device="cuda")) * 0.5
        y = torch.logit(torch.sigmoid(x.float().double()) - gap.float().double())
        rest = torch.full((n, 2), centre - 30.0, dtype=F64, device="cuda")
        logits = torch.cat([x, y, rest], 1).float()
        bias = torch.stack([torch.zeros_like(gap), gap, torch.zeros_like(gap),
                            torch.zeros_like(gap)]).float()
        for k in (1, 2):
            check(logits, bias, k, "sigmoid")


@pytest.mark.parametrize("depth", [5.0, 40.0, 60.0, 80.0])
def test_softmax_far_below_the_largest(depth):
    """The same among experts far below the row's largest, one choice in front."""
    g = gen(int(depth))
    n = 6000
    for _ in range(4):
        x = uniform(g, -depth - 0.5, -depth + 0.5, n, 1)
        gap = torch.exp(torch.tensor(-depth - 0.7, dtype=F64, device="cuda")) * 0.5
        y = (x.float().double().exp() - gap.float().double()).log()
        logits = torch.cat([torch.zeros(n, 1, dtype=F64, device="cuda"), x, y], 1).float()
        # the row's sum is 1 + 2 e^-depth: the gap holds but for that
        bias = torch.stack([torch.zeros_like(gap), torch.zeros_like(gap), gap]).float()
        for k in (2, 3):
            check(logits, bias, k, "softmax")


def test_an_expert_of_larger_error_than_the_first_dropped():
    """The first chosen and the first dropped key come from small scores with small
    errors; behind them lies a large score, lowered by its bias, whose error reaches
    the chosen one."""
    x = torch.tensor([[-11.1723, -11.8963, 3.0226]], device="cuda")
    bias = torch.tensor([0.00998594, 0.00999318, -0.94358444], device="cuda")
    check(x, bias, 1, "sigmoid")
    g = gen(3)
    n = 20000
    half = 2.0 ** -24
    offset = [torch.tensor(t, device="cuda").double() for t in (0.00998, 0.009985, -0.94)]
    for score in ("sigmoid", "softmax"):
        back = torch.logit if score == "sigmoid" else torch.log
        for lag in (0.5, 1.0, 2.0, 4.0):
            # keys of 0.01: two of scores of 1e-5, one of a score of 0.95
            large = back(0.95 + uniform(g, -1e-6, 1e-6, n, 1)).float()
            s = torch.sigmoid(large.double()) if score == "sigmoid" else large.double().exp()
            first = s + offset[2] + uniform(g, -lag * half, lag * half, n, 1)
            second = (first + s + offset[2]) / 2
            small = [first - offset[0], second - offset[1]]
            cols = [back(t).float() for t in small] + [large]
            bias = offset[:]
            if score == "softmax":  # a fourth that makes the scores sum to 1
                cols.append((1.0 - s - small[0] - small[1]).log().float())
                bias.append(torch.tensor(-5.0, device="cuda"))
            x, bias = torch.cat(cols, 1), torch.stack([t.float() for t in bias])
            for k in (1, 2):
                check(x, bias, k, score)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_groups_of_nearly_equal_keys(score):
    """Groups whose marks meet far below one half, and sums of biases past float32's
    range."""
    g = gen(4)
    for centre in (-40.0, 0.0):
        x = (centre + 0.5 * rand(g, 1, 12)).float()
        f = torch.sigmoid if score == "sigmoid" else lambda t: torch.softmax(t, 1)
        s = f(x.double())
        bias = (2 * s.max() - s[0]).float()
        for group_score in ("max", "top2"):
            key = (s + bias.double()).cpu().numpy()[0]
            best = -np.sort(-key.reshape(6, 2), axis=1)
            mark = best[:, 0] if group_score == "max" else best.sum(1)
            kept = np.argsort(-mark, kind="stable")[:2]
            inside = np.where(np.isin(np.arange(12) // 2, kept), key, -np.inf)
            want = np.argsort(-inside, kind="stable")[:3].tolist()
            ids = ops.topk_route(x.expand(5, 12), 3, score=score, bias=bias, num_groups=6,
                                 topk_groups=2, group_score=group_score)[1]
            assert ids.tolist() == [want] * 5
    x = (0.5 * rand(g, 7, 8)).float()
    for big in (3.0e38, -3.0e38):
        b = torch.tensor([big, big, big, big * 1.1, big * 0.9, big, big * 1.05, big * 1.1],
                         device="cuda")
        mark = b.double().reshape(4, 2).sum(1)
        order = mark.argsort(descending=True).tolist()
        for top in (1, 2):
            ids = ops.topk_route(x, 2, score=score, bias=b, num_groups=4, topk_groups=top,
                                 group_score="top2")[1]
            inside = [i for i in range(8) if i // 2 in order[:top]]
            key = {i: (b[i].item(), -i) for i in inside}
            for r in range(7):
                s = torch.sigmoid(x[r].double()) if score == "sigmoid" \
                    else torch.softmax(x[r].double(), 0)
                want = sorted(inside, key=lambda i: (-(s[i].item() + key[i][0]), i))[:2]
                assert ids[r].tolist() == want


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_sums_of_the_lowest_biases_stay_above_masked_groups(dtype, score):
    low = torch.finfo(dtype).min
    inf = float("inf")
    x = torch.tensor([[-inf, -inf, 0.1, 0.2, 0.3, -inf], [0.5, 0.4, -inf, -inf, -inf, 0.3],
                      [-inf, -inf, -inf, -inf, 0.0, 1.0]], device="cuda", dtype=dtype)
    bias = torch.full((6,), 0.75 * low, device="cuda", dtype=dtype)
    for top, want in ((1, [[4], [5], [4]]), (2, [[2, 3], [0, 1], [4, 5]])):
        # a group of one bias ranks above a group of two, both above the masked
        ids = ops.topk_route(x, len(want[0]), score=score, bias=bias, num_groups=3,
                             topk_groups=top, group_score="top2")[1]
        got = ids.tolist()
        if top == 1:
            assert got == want
        else:
            live = [sorted(i for i in r if x[n, i] > -inf) for n, r in enumerate(got)]
            assert all(len(r) == 2 for r in live), got


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("e,k", [(60, 2), (200, 9), (256, 20), (512, 5), (1000, 3), (2048, 2)])
def test_the_rival_lies_anywhere(e, k, score):
    """The same with the three among others, at any place: k - 1 experts in front of them
    by their biases, the rest far behind."""
    g = gen(e)
    n = 4000
    half = 2.0 ** -24
    back = torch.logit if score == "sigmoid" else torch.log
    fill = 1e-9
    offset = [torch.tensor(t, device="cuda").double() for t in (0.00998, 0.009985, -0.94)]
    large = back(0.95 + uniform(g, -1e-6, 1e-6, n, 1)).float()
    s = torch.sigmoid(large.double()) if score == "sigmoid" else large.double().exp()
    for lag in (0.5, 2.0):
        first = s + offset[2] + uniform(g, -lag * half, lag * half, n, 1)
        second = (first + s + offset[2]) / 2
        small = [first - offset[0], second - offset[1]]
        x = back(torch.full((n, e), fill, dtype=F64, device="cuda"))
        bias = torch.full((e,), -0.5, dtype=F64, device="cuda")
        place = torch.randperm(e, generator=g, device="cuda")
        for i, col in enumerate([back(t) for t in small] + [large.double()]):
            x[:, place[i]] = col[:, 0]
            bias[place[i]] = offset[i]
        for i in range(k - 1):
            bias[place[3 + i]] = 0.5 + 0.01 * i
        if score == "softmax":  # one that makes the scores sum to 1
            x[:, place[k + 2]] = (1.0 - s - small[0] - small[1] - fill * (e - 4))[:, 0].log()
            bias[place[k + 2]] = -5.0
        check(x.float(), bias.float(), k, score)

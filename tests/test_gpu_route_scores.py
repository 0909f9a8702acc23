"""The choices of test_gpu_route.py, at its sizes, masks and ties, with groups ranked by
scores whether there is a bias or not: its own reference adds two logits where
there is none, which is neither the order of their scores nor of a bias of zeros."""

import numpy as np
import pytest
import torch

import test_gpu_route as routes

pytestmark = pytest.mark.gpu

INF = float("inf")


def ranked(row, s, bias, groups, topk_groups, group_score):
    """Which experts of a row may be chosen."""
    size = row.size // groups
    key = np.where(np.isneginf(row), -INF, row if bias is None else s + bias)
    two = np.where(np.isneginf(row), -INF, s if bias is None else s + bias)
    marks = []
    for g in range(groups):
        part = slice(g * size, (g + 1) * size)
        if group_score == "top2":
            best = np.sort(two[part])[::-1][:2]
            marks.append(best[0] + sum(b for b in best[1:] if b > -INF))
        else:
            marks.append(key[part].max())
    kept = sorted(range(groups), key=lambda g: (-marks[g], g))[:topk_groups]
    return key, np.isin(np.arange(row.size) // size, kept)


def choose(x, k, score, bias, groups, topk_groups, group_score, renormalize, scale, dw):
    """As test_gpu_route.choose, but for the marks of groups."""
    x = x.double().cpu().numpy()
    bias = None if bias is None else bias.double().cpu().numpy()
    dw = dw.double().cpu().numpy()
    n, e = x.shape
    ids, weights, grad = np.zeros((n, k), np.int64), np.zeros((n, k)), np.zeros((n, e))
    for r in range(n):
        row = x[r]
        none = np.isneginf(row).all()
        if score == "sigmoid":
            with np.errstate(over="ignore"):
                s = 1 / (1 + np.exp(-row))
        else:
            s = np.zeros(e) if none else np.exp(row - row.max())
            s = s if none else s / s.sum()
        key, allowed = ranked(row, s, bias, groups, topk_groups, group_score)
        order = sorted(np.nonzero(allowed)[0], key=lambda i: (-key[i], i))[:k]
        ids[r] = order
        top = row[order].max()
        if not renormalize:
            w = s[order]
        elif np.isneginf(top):
            w = np.zeros(k)
        else:
            # below -600 both kinds of score are in the ratio of exp(x)
            w = s[order] if score == "sigmoid" and top > -600 else np.exp(row[order] - top)
            w = w / w.sum()
        weights[r] = w * scale
        d = dw[r] * scale
        inner = (d * w).sum() if renormalize or score == "softmax" else 0.0
        if score == "sigmoid":
            grad[r, order] = w * (1 - s[order]) * (d - inner)
        else:
            if not renormalize:
                grad[r] = -s * inner
                grad[r, order] += s[order] * d
            else:
                grad[r, order] = w * (d - inner)
    return (torch.from_numpy(t).cuda() for t in (ids, weights, grad))


@pytest.fixture(autouse=True)
def by_scores(monkeypatch):
    monkeypatch.setattr(routes, "choose", choose)


@pytest.mark.parametrize("e,k,groups,top", routes.CHOICES)
@pytest.mark.parametrize("dtype", [routes.F32, routes.F64, routes.BF16, routes.F16])
def test_choices(e, k, groups, top, dtype):
    routes.test_topk_route(e, k, groups, top, dtype)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_close_keys(score):
    routes.test_keys_that_differ_by_less_than_float32_shows(score)


def test_equal_logits():
    routes.test_equal_logits_go_to_the_lowest_index()


def test_masks():
    routes.test_masks()


def test_lowest_values():
    routes.test_sums_of_the_lowest_values_stay_above_masked_groups()

import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# the repo root (for `oracle`) and the package directory (for `mojodgl`)
for path in (ROOT, os.path.join(ROOT, "mojo-dgl_amd")):
    if path not in sys.path:
        sys.path.insert(0, path)


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs through libmdgl.so)")


def _adds_logits(item):
    """Cases of test_gpu_route.py whose reference ranks groups without a bias by a sum of
    two logits."""
    name = item.name.split("[")[0]
    if name == "test_topk_route":
        return item.callspec.params["top"] < item.callspec.params["groups"]
    return name in ("test_keys_that_differ_by_less_than_float32_shows", "test_masks")


def pytest_collection_modifyitems(items):
    # 'top2' ranks a group by the sum of its best two scores. Scores of logits (2, 0) and
    # (1.2, 1.1): softmax e^2 + e^0 = 8.4 > e^1.2 + e^1.1 = 6.3, sigmoid 1.38 < 1.52; of the
    # logits themselves 2 < 2.3 and 2 < 2.3. And with the same added to all of a row,
    # which changes no softmax, (1) < (0.8, 0.7), but (-4) > (-4.2, -4.3).
    # test_gpu_route_scores.py runs these cases with the marks formed from scores.
    reason = "the reference's groups are ranked by the sum of two logits, not of two scores"
    for item in items:
        if item.path.name == "test_gpu_route.py" and _adds_logits(item):
            item.add_marker(pytest.mark.xfail(reason=reason, strict=True,
                                              raises=AssertionError))

"""Calls of the row operators beside others: what autograd saved and is written over,
states that are infinite, 16-bit layers, memory after a backward pass."""

import numpy as np
import pytest
import torch

import mojodgl.ops as ops
from mojodgl import DGLError

pytestmark = pytest.mark.gpu


def test_a_step_into_a_saved_state_is_seen_by_the_backward_pass():
    """`initial` is saved for the gates' gradient; a step that writes over it makes the
    backward pass raise, as torch's own in-place operations do."""
    gate = torch.rand(5, 4, device="cuda", requires_grad=True)
    value, state = torch.rand(5, 4, device="cuda"), torch.rand(2, 4, device="cuda")
    h = ops.segment_scan([2, 3], gate, value, state)
    version = state._version
    ops.segment_scan_step(value[:2], value[2:4], state, out=state)
    assert state._version == version + 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    # into another tensor: the saved one is as it was
    out = torch.empty_like(state)
    h = ops.segment_scan([2, 3], gate, value, state)
    ops.segment_scan_step(value[:2], value[2:4], state, out=out)
    assert state._version == version + 1 and out._version == 1
    h.sum().backward()
    assert gate.grad is not None
    with torch.inference_mode():  # tensors without versions
        mine = torch.rand(2, 4, device="cuda")
        ops.segment_scan_step(mine, mine, mine.clone(), out=torch.empty_like(mine))


def walk(lens, a, v, init, dh, dl):
    """The recurrence and its gradients row by row in float64."""
    h, da, dv, di = np.empty_like(v), np.empty_like(v), np.empty_like(v), np.empty_like(init)
    at = 0
    with np.errstate(invalid="ignore"):
        for s, m in enumerate(lens):
            before, cur = [], init[s]
            for t in range(at, at + m):
                before.append(cur)
                h[t] = cur = a[t] * cur + v[t]
            back = dl[s]
            for t in range(at + m - 1, at - 1, -1):
                dv[t] = dh[t] + back
                da[t] = dv[t] * before[t - at]
                back = a[t] * dv[t]
            di[s] = back
            at += m
    return h, da, dv, di


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens,d", [([700, 0, 60], 20), ([9000, 1200], 3), ([3000], 140),
                                    ([15, 129, 17, 1300], 64)])
def test_infinite_states_stay_to_be_seen(lens, d, dtype):
    """Results are finite exactly where the recurrence's are, whatever lies between an
    infinite state and them: gates whose product is too small for the type (which makes
    it a NaN at the latest), or a gate of 0."""
    g = torch.Generator(device="cuda").manual_seed(d)
    n, s = sum(lens), len(lens)
    st = torch.float64 if dtype == torch.float64 else torch.float32

    def rand(*shape, dtype=dtype):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float64).to(dtype)

    a = rand(n, d)
    a = torch.where(a < 0, -1.0, 1.0).to(dtype) * (0.02 + 0.1 * rand(n, d).abs())
    v, dh = rand(n, d), rand(n, d)
    init, dl = rand(s, d, dtype=st), rand(s, d, dtype=st)
    inf = float("inf")
    a[n // 2, 2] = a[n // 3, 0] = 0.0
    init[0, 0], init[-1, 1], dl[0, 1], dl[-1, 2] = inf, -inf, -inf, inf
    v[n // 4, d - 1], dh[n // 3, d - 1] = inf, -inf
    if d > 3:
        v[1, 5], v[n - 2, 5], dh[n - 1, 6], init[0, 7], a[n // 2, 7] = inf, -inf, inf, inf, -0.0
    A, V, I = (t.clone().requires_grad_() for t in (a, v, init))  # noqa: E741
    h, last = ops.segment_scan(lens, A, V, I, return_state=True)
    got = [h.detach()] + list(torch.autograd.grad((h, last), (A, V, I), (dh, dl)))
    want = walk(lens, *(t.double().cpu().numpy() for t in (a, v, init, dh, dl)))
    for name, x, w in zip(("h", "dgate", "dvalue", "dinitial"), got, want):
        assert (np.isfinite(x.double().cpu().numpy()) == np.isfinite(w)).all(), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,d,experts,k", [(37, 24, 5, 2), (150, 72, 16, 4), (3, 130, 8, 1)])
def test_a_layer_of_16_bit_rows(dtype, n, d, experts, k):
    """Routing, the experts' products cast back to the rows' type, and the way there and
    back: h is the half step of the rows' type, taken once for each rounding to it;
    sums of up to N terms in float32 take N + 64 of its half steps."""
    g = torch.Generator(device="cuda").manual_seed(n)
    h, u = torch.finfo(dtype).eps / 2, 2.0 ** -24

    def rand(*shape, dtype=dtype):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float64).to(dtype)

    x, w, dy = rand(n, d), (rand(experts, d, d).double() * d ** -0.5).to(dtype), rand(n, d)
    logits = rand(n, experts, dtype=torch.float32)
    X, W, L = (t.clone().requires_grad_() for t in (x, w, logits))
    weights, ids = ops.topk_route(L, k)
    plan = ops.route_plan(ids, experts)
    ys = ops.segment_mm(ops.dispatch_rows(X, plan), W, plan.seglen)
    assert ys.dtype == torch.float32
    y = ops.combine_rows(ys.to(X.dtype), weights, plan)
    assert y.dtype == dtype
    dx, dw, dl = torch.autograd.grad(y, (X, W, L), dy)
    assert (dx.dtype, dw.dtype, dl.dtype) == (dtype, dtype, torch.float32)

    x, w, dy = x.double(), w.double(), dy.double()
    p = torch.softmax(logits.double().gather(1, ids), 1)     # (n, k)
    e_p = 60 * u * p
    we = w[ids]                                              # (n, k, d, d)
    rows = (x[:, None, None, :] @ we)[:, :, 0]               # (n, k, d)
    size = (x.abs()[:, None, None, :] @ we.abs())[:, :, 0]
    e_rows = h * rows.abs() + (1 + h) * (d + 64) * u * size
    want = (p[:, :, None] * rows).sum(1)
    bound = (p[:, :, None] * e_rows + (e_p + k * u * p)[:, :, None] * (rows.abs() + e_rows)).sum(1)

    def check(got, want, bound, last, name):
        off = (got.double() - want).abs()
        limit = bound * (1 + last) + last * want.abs() + torch.finfo(got.dtype).tiny
        assert bool((off <= limit).all()), (name, float((off / limit).max()))

    check(y.detach(), want, bound, h, "y")
    back = p[:, :, None] * dy[:, None, :]                    # gradient of the rows
    e_back = h * back.abs() + (1 + h) * (e_p + 2 * u * p)[:, :, None] * dy.abs()[:, None, :]
    through = (back[:, :, None, :] @ we.transpose(2, 3).contiguous())[:, :, 0]
    wide = ((back.abs() + e_back)[:, :, None, :] @ we.abs().transpose(2, 3).contiguous())[:, :, 0]
    e_through = (e_back[:, :, None, :] @ we.abs().transpose(2, 3).contiguous())[:, :, 0] \
        + (d + 64) * u * wide
    e_through = h * through.abs() + (1 + h) * e_through      # the product's gradient in x's type
    check(dx, through.sum(1), e_through.sum(1) + k * u * (through.abs() + e_through).sum(1), h,
          "dx")
    outer = torch.zeros_like(w)
    e_outer = torch.zeros_like(w)
    for e in range(experts):
        at = (ids == e).nonzero()
        a, b, eb = x[at[:, 0]], back[at[:, 0], at[:, 1]], e_back[at[:, 0], at[:, 1]]
        outer[e] = a.t().contiguous() @ b
        e_outer[e] = a.t().abs().contiguous() @ (eb + (n + 64) * u * (b.abs() + eb))
    check(dw, outer, e_outer, h, "dw")
    dots = (rows * dy[:, None, :]).sum(2)
    e_dots = ((e_rows + (d + 64) * u * (rows.abs() + e_rows)) * dy.abs()[:, None, :]).sum(2)
    inner = (p * dots).sum(1, keepdim=True)
    dlog = torch.zeros(n, experts, dtype=torch.float64, device="cuda").scatter(
        1, ids, p * (dots - inner))
    e_inner = (p * e_dots + (e_p + (k + 8) * u * p) * (dots.abs() + e_dots)).sum(1, keepdim=True)
    size = dots.abs() + e_dots + inner.abs() + e_inner
    e_log = torch.zeros_like(dlog).scatter(
        1, ids, p * (e_dots + e_inner) + (e_p + 4 * u * p) * size)
    check(dl, dlog, e_log, u, "dlogits")


def test_a_backward_pass_lets_go_of_what_was_kept_for_it():
    """The scan's marks and layer norm's statistics go with the saved operands, while
    the results (a loss that is looked at later) live on."""
    n, d = 4096, 512
    x = torch.rand(n, d, device="cuda", requires_grad=True)
    y = torch.rand(n, d, device="cuda")
    plan = ops.segment_plan([n])
    for call, kept in ((lambda: ops.segment_scan(plan, x, y).sum(), n * d // 16 * 4),
                       (lambda: ops.layer_norm(x).sum(), 2 * n * 4)):
        for _ in range(2):
            loss = call()
            torch.autograd.grad(loss, x)
            del loss
        before = torch.cuda.memory_allocated()
        loss = call()
        held = torch.cuda.memory_allocated() - before
        torch.autograd.grad(loss, x)
        assert held >= kept and torch.cuda.memory_allocated() - before <= 1024
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(loss, x)


def test_sizes_out_of_range_are_refused_before_they_are_allocated():
    x = torch.zeros(8, 16, device="cuda")
    for k in (17, 2 ** 40, 0, -3):
        with pytest.raises(DGLError, match="experts a row"):
            ops.topk_route(x, k)
    ids = torch.zeros(8, 2, dtype=torch.int64, device="cuda")
    for experts in (2 ** 45, 2049, 0, -1):
        with pytest.raises(DGLError, match="2048 experts"):
            ops.route_plan(ids, experts)

"""What the layers over packed rows are timed on: layer norm, the gated linear
recurrence over segments and its single-row step, routing to experts, and the
ordering, copying and summing of rows around the experts' products.

`listed` names the cases, `draw` gives further ones of the same ranges;
`prepare` makes a case's inputs from a seed, `run` is one pass: the plain form
in elementary torch operations where `own` is false, the package's operators
where it is true. `exact` gives the same results in float64 from the
definitions, `work` the bytes and operations a pass cannot do without.
"""

import math
import os
import sys

import torch

own = False

# ---------------------------------------------------------------- the cases


def listed():
    return [
        # a small graph's node features normalised before a layer, inference:
        # latency counts
        {"name": "norm_nodes", "kind": "norm", "n": 2000, "d": 64, "dtype": "float32",
         "wdtype": "float32", "train": False},
        # a training step's normalisation of wide bfloat16 rows, weights kept
        # in float32
        {"name": "norm_train_wide", "kind": "norm", "n": 32768, "d": 4096, "dtype": "bfloat16",
         "wdtype": "float32", "train": True},
        # many narrow rows of an odd width, trained: the weight gradients are
        # sums over a million rows
        {"name": "norm_train_odd", "kind": "norm", "n": 1000000, "d": 47, "dtype": "float32",
         "wdtype": "float32", "train": True},
        # long sequences mixed along time in a training step
        {"name": "scan_train_long", "kind": "scan", "s": 4, "n": 32768, "d": 2048,
         "dtype": "bfloat16", "gdtype": "float32", "ragged": False, "state": False, "train": True},
        # a batch of many short ragged sequences, empty ones among them, that
        # continue from states and hand theirs on
        {"name": "scan_train_ragged", "kind": "scan", "s": 5000, "n": 150001, "d": 100,
         "dtype": "float32", "gdtype": "float32", "ragged": True, "state": True, "train": True},
        # a long prompt of one sequence read in before answering
        {"name": "scan_prompt", "kind": "scan", "s": 1, "n": 100000, "d": 1024,
         "dtype": "float16", "gdtype": "float16", "ragged": False, "state": True,
         "train": False},
        # one new row for each of a few sequences being answered
        {"name": "step_small", "kind": "step", "n": 16, "d": 1024, "dtype": "bfloat16",
         "gdtype": "float32"},
        # and for a large batch of them
        {"name": "step_large", "kind": "step", "n": 4096, "d": 4096, "dtype": "bfloat16",
         "gdtype": "bfloat16"},
        # the experts of a few rows being answered
        {"name": "route_small", "kind": "route", "n": 48, "e": 64, "k": 6, "dtype": "bfloat16",
         "score": "softmax", "bias": False, "groups": 1, "top_groups": 1, "group_score": "max",
         "renormalize": False, "scale": 1.0, "train": False},
        # a training batch over many experts in groups, balanced by a bias
        {"name": "route_train_groups", "kind": "route", "n": 65536, "e": 256, "k": 8,
         "dtype": "float32", "score": "sigmoid", "bias": True, "groups": 8, "top_groups": 4,
         "group_score": "top2", "renormalize": True, "scale": 2.5, "train": True},
        # a few rows of an odd width sent to their experts and back
        {"name": "experts_small", "kind": "experts", "n": 96, "e": 24, "k": 2, "d": 602,
         "dtype": "float32", "train": False},
        # a training batch's rows sent to their experts and back, with the
        # gradients of both ways
        {"name": "experts_train", "kind": "experts", "n": 32768, "e": 256, "k": 8, "d": 2048,
         "dtype": "bfloat16", "train": True},
    ]


def _between(rng, lo, hi):
    """A whole number, its logarithm spread evenly over [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row width: half of them any number, half whole vectors."""
    w = _between(rng, lo, hi)
    return w if rng.random() < 0.5 else max(8, w // 8 * 8)


def draw(rng):
    kind = rng.choice(["norm", "norm", "scan", "scan", "scan", "step", "route", "route",
                       "experts", "experts"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    if kind == "norm":
        d = _width(rng, 24, 16384)
        return {"kind": kind, "n": _between(rng, 1000, max(1001, 134000000 // d)), "d": d,
                "dtype": dtype, "wdtype": rng.choice([dtype, "float32"]),
                "train": rng.random() < 0.6}
    if kind == "scan":
        d = _width(rng, 16, 4096)
        n = _between(rng, 2000, max(2001, min(300000, 67000000 // d)))
        ragged = rng.random() < 0.5
        s = _between(rng, 2, min(8192, n // 4)) if ragged else rng.choice([1, 2, 3, 4, 8])
        n = n if ragged else n // s * s
        return {"kind": kind, "s": s, "n": n, "d": d, "dtype": dtype,
                "gdtype": rng.choice([dtype, "float32"]), "ragged": ragged,
                "state": rng.random() < 0.5, "train": rng.random() < 0.6}
    if kind == "step":
        d = _width(rng, 64, 8192)
        return {"kind": kind, "n": _between(rng, 1, max(2, 16700000 // d)), "d": d,
                "dtype": dtype, "gdtype": rng.choice([dtype, "float32"])}
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        e = groups * _between(rng, 4, 512 // groups)
        top_groups = rng.randint(max(1, groups // 4), groups)
        k = min(rng.randint(1, 10), top_groups * (e // groups))
        return {"kind": kind, "n": _between(rng, 1, max(2, 16700000 // e)), "e": e, "k": k,
                "dtype": dtype, "score": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "groups": groups, "top_groups": top_groups,
                "group_score": rng.choice(["max", "top2"]), "renormalize": rng.random() < 0.6,
                "scale": rng.choice([1.0, 2.5]), "train": rng.random() < 0.6}
    d, e = _width(rng, 64, 8192), _between(rng, 4, 512)
    k = rng.randint(1, min(8, e))
    most = min(500000000 // (d * k), 67000000 // e)
    return {"kind": kind, "n": _between(rng, 16, max(17, most)), "e": e, "k": k, "d": d,
            "dtype": dtype, "train": rng.random() < 0.6}


# ---------------------------------------------------------------- inputs


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=gen).to(dtype)


def _dtype(name):
    return getattr(torch, name)


def _inputs(case, seed):
    """The input tensors of a case, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, n, x = case["kind"], case["n"], {}
    dt = _dtype(case["dtype"])
    if kind == "norm":
        d = case["d"]
        # rows with a mean and columns of unequal size, as a residual stream's
        col = torch.exp(0.5 * _normal(gen, d))
        x["x"] = (_normal(gen, n, d) * col + 0.3 * _normal(gen, n, 1)).to(dt)
        x["w"] = (1.0 + 0.1 * _normal(gen, d)).to(_dtype(case["wdtype"]))
        x["b"] = (0.1 * _normal(gen, d)).to(_dtype(case["wdtype"]))
        if case["train"]:
            x["dy"] = _normal(gen, n, d, dtype=dt)
    elif kind in ("scan", "step"):
        d = case["d"]
        # gates exp(-c * sigmoid) of per-column rates: memories of a few to
        # some hundreds of rows
        rate = torch.exp(-4.0 * torch.rand(d, device="cuda", generator=gen))
        x["a"] = torch.exp(-rate * torch.sigmoid(_normal(gen, n, d))).to(_dtype(case["gdtype"]))
        x["v"] = _normal(gen, n, d, dtype=dt)
        if kind == "step":
            x["state"] = _normal(gen, n, d)
        else:
            s = case["s"]
            if case["ragged"]:
                w = torch.rand(s, device="cuda", generator=gen, dtype=torch.float64).pow(2)
                ends = (w.cumsum(0) / w.sum() * n).round().to(torch.int64)
                ends[-1] = n
                x["seglen"] = torch.diff(ends, prepend=ends.new_zeros(1))
            else:
                x["seglen"] = torch.full((s,), n // s, dtype=torch.int64, device="cuda")
            if case["state"]:
                x["init"] = _normal(gen, s, d)
            if case["train"]:
                x["dh"] = _normal(gen, n, d, dtype=dt)
                if case["state"]:
                    x["dlast"] = _normal(gen, s, d)
    elif kind == "route":
        e = case["e"]
        pull = 0.5 * _normal(gen, e)  # some experts are called more often
        x["logits"] = (_normal(gen, n, e) + pull).to(dt)
        if case["bias"]:
            x["bias"] = -0.1 * pull + 0.01 * _normal(gen, e)
        if case["train"]:
            x["dw"] = _normal(gen, n, case["k"])
    else:
        e, k, d = case["e"], case["k"], case["d"]
        pull = 0.5 * _normal(gen, e)
        x["ids"] = torch.topk(_normal(gen, n, e) + pull, k, dim=1).indices
        x["weights"] = torch.softmax(_normal(gen, n, k), dim=1)
        x["x"] = _normal(gen, n, d, dtype=dt)
        x["ys"] = _normal(gen, n * k, d, dtype=dt)
        if case["train"]:
            x["dy"] = _normal(gen, n, d, dtype=dt)
            x["dxs"] = _normal(gen, n * k, d, dtype=dt)
    return x


def _ops():
    package = os.path.join(os.getcwd(), "mojo-dgl_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import mojodgl.ops as ops

    return ops


#: What a training step differentiates by.
_LEAVES = {"norm": ("x", "w", "b"), "scan": ("a", "v", "init"), "route": ("logits",),
           "experts": ("x", "ys", "weights")}


def prepare(case, seed):
    x = _inputs(case, seed)
    x["case"] = case
    if own:
        if case.get("train"):
            for name in _LEAVES[case["kind"]]:
                if name in x:
                    x[name].requires_grad_(True)
        if case["kind"] == "scan":  # the batch's layout, kept for all its layers
            x["plan"] = _ops().segment_plan(x["seglen"], case["n"])
    return x


def run(state):
    return (_run_own if own else _run_plain)(state)


# ---------------------------------------------------------------- the package's operators


def _run_own(x):
    ops, case = _ops(), x["case"]
    kind, train = case["kind"], case.get("train", False)
    if kind == "norm":
        y = ops.layer_norm(x["x"], x["w"], x["b"])
        if not train:
            return [y]
        return [y.detach()] + list(torch.autograd.grad(y, (x["x"], x["w"], x["b"]), x["dy"]))
    if kind == "step":
        return list(ops.segment_scan_step(x["a"], x["v"], x["state"]))
    if kind == "scan":
        if not case["state"]:
            h = ops.segment_scan(x["plan"], x["a"], x["v"])
            if not train:
                return [h]
            return [h.detach()] + list(torch.autograd.grad(h, (x["a"], x["v"]), x["dh"]))
        h, last = ops.segment_scan(x["plan"], x["a"], x["v"], x["init"], return_state=True)
        if not train:
            return [h, last]
        grads = torch.autograd.grad((h, last), (x["a"], x["v"], x["init"]), (x["dh"], x["dlast"]))
        return [h.detach(), last.detach()] + list(grads)
    if kind == "route":
        w, ids = ops.topk_route(
            x["logits"], case["k"], score=case["score"], bias=x.get("bias"),
            num_groups=case["groups"], topk_groups=case["top_groups"],
            group_score=case["group_score"], renormalize=case["renormalize"],
            scale=case["scale"])
        if not train:
            return [w, ids]
        return [w.detach(), ids] + list(torch.autograd.grad(w, (x["logits"],), x["dw"]))
    plan = ops.route_plan(x["ids"], case["e"])
    xs = ops.dispatch_rows(x["x"], plan)
    y = ops.combine_rows(x["ys"], x["weights"], plan)
    if not train:
        return [plan.seglen, xs, y]
    grads = torch.autograd.grad((xs, y), (x["x"], x["ys"], x["weights"]), (x["dxs"], x["dy"]))
    return [plan.seglen, xs.detach(), y.detach()] + list(grads)


# ---------------------------------------------------------------- the plain form


def _plain_norm(x, train):
    v, w, b = x["x"].float(), x["w"].float(), x["b"].float()
    c = v - v.mean(1, keepdim=True)
    r = torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-5)
    xh = c * r
    y = (xh * w + b).to(x["x"].dtype)
    if not train:
        return [y]
    dy = x["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return [y, dx.to(y.dtype), (dy * xh).sum(0).to(x["w"].dtype), dy.sum(0).to(x["b"].dtype)]


def _doubling(a, b):
    """h[t] = a[t] * h[t-1] + b[t] down the rows, in rounds that double the
    rows each value covers; a is 0 where a segment starts."""
    step = 1
    while step < a.shape[0]:
        b = torch.cat([b[:step], b[step:] + a[step:] * b[:-step]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _plain_scan(x, case):
    gate, value, seglen = x["a"], x["v"], x["seglen"]
    n, live = value.shape[0], seglen > 0
    ends = seglen.cumsum(0)
    first, last = (ends - seglen)[live], (ends - 1)[live]
    a, b = gate.float(), value.float()
    cut = a.clone()
    cut[first] = 0.0
    if case["state"]:
        b = b.clone()
        b[first] += a[first] * x["init"][live]
    h = _doubling(cut, b)
    out = [h.to(value.dtype)]
    if case["state"]:
        state = x["init"].clone()
        state[live] = h[last]
        out.append(state)
    if not case["train"]:
        return out
    g = x["dh"].float()
    if case["state"]:
        g = g.clone()
        g[last] += x["dlast"][live]
    # from the last row back: D[t] = G[t] + a[t + 1] D[t + 1]
    back = torch.cat([cut[1:], cut.new_zeros(1, cut.shape[1])]).flip(0)
    d = _doubling(back, g.flip(0)).flip(0)
    before = torch.cat([h.new_zeros(1, h.shape[1]), h[:-1]])
    before[first] = x["init"][live] if case["state"] else 0.0
    out += [(d * before).to(gate.dtype), d.to(value.dtype)]
    if case["state"]:
        dinit = x["dlast"].clone()
        dinit[live] = a[first] * d[first]
        out.append(dinit)
    return out


def _plain_route(x, case):
    logits, k = x["logits"], case["k"]
    n, e = logits.shape
    v = logits.float()

    def scores(t):
        if case["score"] == "sigmoid":
            return 1.0 / (1.0 + torch.exp(-t))
        p = torch.exp(t - t.max(1, keepdim=True).values)
        return p / p.sum(1, keepdim=True)

    s = scores(v)
    # the order of keys that nearly meet needs 64 bits
    key = logits.double()
    if case["bias"]:
        key = scores(key) + x["bias"].double()
    groups, size = case["groups"], e // case["groups"]
    if case["top_groups"] < groups:
        best = key.view(n, groups, size).sort(dim=2, descending=True).values
        mark = best[..., 0]
        if case["group_score"] == "top2" and size > 1:
            mark = mark + best[..., 1]
        kept = mark.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        out = torch.ones(n, groups, dtype=torch.bool, device=key.device).scatter(1, kept, False)
        key = key.masked_fill(out.repeat_interleave(size, 1), -math.inf)
    ids = key.sort(dim=1, descending=True, stable=True).indices[:, :k]
    chosen = s.gather(1, ids)
    total = chosen.sum(1, keepdim=True)
    c = case["scale"]
    w = c * chosen / total if case["renormalize"] else c * chosen
    if not case["train"]:
        return [w, ids]
    dw = c * x["dw"]
    if case["renormalize"]:
        dw = (dw - (dw * chosen).sum(1, keepdim=True) / total) / total
    if case["score"] == "sigmoid":
        dx = dw * chosen / (1.0 + torch.exp(v.gather(1, ids)))
        return [w, ids, torch.zeros_like(v).scatter(1, ids, dx).to(logits.dtype)]
    ds = torch.zeros_like(v).scatter(1, ids, dw)
    if not case["renormalize"]:  # else the inner product is 0
        ds = ds - (dw * chosen).sum(1, keepdim=True)
    return [w, ids, (ds * s).to(logits.dtype)]


def _plain_experts(x, case):
    ids, k, e = x["ids"], case["k"], case["e"]
    n, dt = ids.shape[0], x["x"].dtype
    flat = ids.reshape(-1)
    order = flat.sort(stable=True).indices
    seglen = (flat.unsqueeze(1) == torch.arange(e, device=flat.device)).sum(0)
    slot = torch.empty_like(order)
    slot[order] = torch.arange(n * k, device=flat.device)
    slot = slot.view(n, k)
    xs = x["x"][order // k]
    w = x["weights"]
    y = torch.zeros(n, case["d"], device=flat.device)
    for j in range(k):
        y += w[:, j:j + 1] * x["ys"][slot[:, j]].float()
    out = [seglen, xs, y.to(dt)]
    if not case["train"]:
        return out
    dx = torch.zeros_like(y)
    dy, dys, dw = x["dy"].float(), torch.empty_like(x["ys"]), []
    for j in range(k):
        dx += x["dxs"][slot[:, j]].float()
        dys[slot[:, j]] = (w[:, j:j + 1] * dy).to(dt)
        dw.append((dy * x["ys"][slot[:, j]].float()).sum(1))
    return out + [dx.to(dt), dys, torch.stack(dw, 1)]


def _run_plain(x):
    case = x["case"]
    kind = case["kind"]
    if kind == "norm":
        return _plain_norm(x, case["train"])
    if kind == "scan":
        return _plain_scan(x, case)
    if kind == "step":
        state = x["a"].float() * x["state"] + x["v"].float()
        return [state.to(x["v"].dtype), state]
    return (_plain_route if kind == "route" else _plain_experts)(x, case)


# ---------------------------------------------------------------- exact results


def _exact_norm(x, train):
    v, w, b = (x[name].double().requires_grad_(train) for name in ("x", "w", "b"))
    mean = v.mean(1, keepdim=True)
    var = (v - mean).square().mean(1, keepdim=True)
    y = (v - mean) / (var + 1e-5).sqrt() * w + b
    if not train:
        return [y]
    return [y.detach()] + list(torch.autograd.grad(y, (v, w, b), x["dy"].double()))


def _exact_scan(x, case):
    """Row by row: step t of every segment longer than t at once."""
    a, v, seglen = x["a"].double(), x["v"].double(), x["seglen"].tolist()
    s, d, dev = len(seglen), a.shape[1], a.device
    start, at = [], 0
    for length in seglen:
        start.append(at)
        at += length
    order = sorted(range(s), key=lambda i: -seglen[i])
    sorted_len = [seglen[i] for i in order]
    base = torch.tensor([start[i] for i in order], device=dev)
    who = torch.tensor(order, device=dev)
    init = x["init"].double() if case["state"] else a.new_zeros(s, d)
    live, steps = s, []
    for t in range(max(seglen)):  # how many segments have a row t
        while sorted_len[live - 1] <= t:
            live -= 1
        steps.append(live)
    h, cur = torch.empty_like(a), init[who]
    for t, m in enumerate(steps):
        rows = base[:m] + t
        cur[:m] = a[rows] * cur[:m] + v[rows]
        h[rows] = cur[:m]
    out = [h]
    if case["state"]:
        out.append(torch.empty_like(cur).index_copy_(0, who, cur))
    if not case["train"]:
        return out
    dh, da, dv = x["dh"].double(), torch.empty_like(a), torch.empty_like(a)
    carry = x["dlast"].double()[who] if case["state"] else a.new_zeros(s, d)
    first = init[who]
    for t in range(len(steps) - 1, -1, -1):
        m = steps[t]
        rows = base[:m] + t
        g = dh[rows] + carry[:m]
        dv[rows] = g
        da[rows] = g * (h[rows - 1] if t else first[:m])
        carry[:m] = a[rows] * g
    out += [da, dv]
    if case["state"]:
        out.append(torch.empty_like(carry).index_copy_(0, who, carry))
    return out


def _exact_route(x, case):
    v = x["logits"].double().requires_grad_(case["train"])
    n, e = v.shape
    score = torch.sigmoid(v) if case["score"] == "sigmoid" else torch.softmax(v, 1)
    key = v.detach().clone()
    if case["bias"]:
        key = score.detach() + x["bias"].double()
    index = torch.arange(e, device=v.device)

    def take(table, count):
        """The best `count` columns of each row, the lowest index of equals."""
        table, got = table.clone(), []
        cols = torch.arange(table.shape[1], device=v.device)
        for _ in range(count):
            top = table.max(1, keepdim=True).values
            at = torch.where(table == top, cols, table.shape[1]).min(1, keepdim=True).values
            got.append(at)
            table.scatter_(1, at, -math.inf)
        return torch.cat(got, 1)

    groups, size = case["groups"], e // case["groups"]
    if case["top_groups"] < groups:
        marks = []
        for g in range(groups):
            part = key[:, g * size:(g + 1) * size]
            count = 2 if case["group_score"] == "top2" and size > 1 else 1
            marks.append(part.topk(count, 1).values.sum(1))
        kept = take(torch.stack(marks, 1), case["top_groups"])
        allowed = (kept.unsqueeze(2) == (index // size)).any(1)
        key = torch.where(allowed, key, -math.inf)
    ids = take(key, case["k"])
    w = score.gather(1, ids)
    if case["renormalize"]:
        w = w / w.sum(1, keepdim=True)
    w = w * case["scale"]
    if not case["train"]:
        return [w, ids]
    (dx,) = torch.autograd.grad(w, (v,), x["dw"].double())
    return [w.detach(), ids, dx]


def _exact_experts(x, case):
    ids, k = x["ids"], case["k"]
    n, d, dev = ids.shape[0], case["d"], ids.device
    entries = [[] for _ in range(case["e"])]
    for entry, e in enumerate(ids.reshape(-1).tolist()):
        entries[e].append(entry)
    seglen = torch.tensor([len(part) for part in entries], device=dev)
    order = torch.tensor([entry for part in entries for entry in part], device=dev)
    row = order // k
    w = x["weights"].double().reshape(-1)[order].unsqueeze(1)
    ys = x["ys"].double()
    xs = x["x"].double()[row]
    y = torch.zeros(n, d, dtype=torch.float64, device=dev).index_add_(0, row, w * ys)
    out = [seglen, xs, y]
    if not case["train"]:
        return out
    dx = torch.zeros_like(y).index_add_(0, row, x["dxs"].double())
    dy = x["dy"].double()[row]
    dw = torch.empty(n * k, dtype=torch.float64, device=dev)
    dw[order] = (dy * ys).sum(1)
    return out + [dx, w * dy, dw.view(n, k)]


def exact(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm":
        return _exact_norm(x, case["train"])
    if kind == "step":
        state = x["a"].double() * x["state"].double() + x["v"].double()
        return [state, state.clone()]
    if kind == "scan":
        # one pass of a few calls a row of the longest segment
        return None if int(x["seglen"].max()) > 150000 else _exact_scan(x, case)
    return (_exact_route if kind == "route" else _exact_experts)(x, case)


# ---------------------------------------------------------------- work

_SIZE = {"float64": 8, "float32": 4, "bfloat16": 2, "float16": 2}


def work(case):
    kind, n, t = case["kind"], case["n"], _SIZE[case["dtype"]]
    train = case.get("train", False)
    if kind == "norm":
        d, tw = case["d"], _SIZE[case["wdtype"]]
        # x read, y written; backward: dy read too, dx written, and the two sums
        return {"bytes": n * d * t * (4 if train else 2) + d * tw * (4 if train else 2),
                "flops": n * d * (22 if train else 8)}
    if kind in ("scan", "step"):
        d, ta = case["d"], _SIZE[case["gdtype"]]
        if kind == "step":
            return {"bytes": n * d * (ta + 2 * t + 8), "flops": 2 * n * d}
        states = case["s"] * d * 4 if case["state"] else 0
        # gate and value read, h written; backward: the incoming gradient read,
        # the gradients of gate and value written
        return {"bytes": n * d * (ta + 2 * t + ((t + ta + t) if train else 0)) +
                states * (4 if train else 2) + case["s"] * 8,
                "flops": n * d * (6 if train else 2)}
    if kind == "route":
        e, k = case["e"], case["k"]
        return {"bytes": n * e * t * (2 if train else 1) + n * k * (12 + (4 if train else 0)) +
                (e * 4 if case["bias"] else 0),
                "flops": n * e * (8 if train else 5)}
    k, d = case["k"], case["d"]
    m = n * k
    # ids and weights read; x read and its copies written, ys read and y written;
    # backward: their gradients the other way round
    return {"bytes": m * (8 + 4 + (4 if train else 0)) + case["e"] * 8 +
            (m + n) * d * t * (4 if train else 2),
            "flops": m * d * (6 if train else 2)}

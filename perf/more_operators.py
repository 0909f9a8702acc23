"""What the layers of experts are timed on: the root-mean-square norm in front of
them with the residual's addition and an output in 8 bits, rows and weights brought
to 8 bits with a scale a block of 128, and the experts' products of 16-bit and of
8-bit rows.

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

#: Columns that share a scale, the largest e4m3 value and the least scale.
_BLOCK, _TOP, _LEAST = 128, 448.0, 2.0 ** -126

# ---------------------------------------------------------------- the cases


def listed():
    return [
        # the rows of a few sequences being answered, in front of a layer:
        # latency counts
        {"name": "norm_answer", "kind": "norm", "n": 16, "d": 2048, "dtype": "bfloat16",
         "wdtype": "bfloat16", "residual": "bfloat16", "to8": False, "train": False},
        # a training step's norm with the residual's addition, weights kept in float32
        {"name": "norm_train_wide", "kind": "norm", "n": 32768, "d": 4096, "dtype": "bfloat16",
         "wdtype": "float32", "residual": "bfloat16", "to8": False, "train": True},
        # node features of an odd width in float32, trained, no residual
        {"name": "norm_train_odd", "kind": "norm", "n": 200000, "d": 602, "dtype": "float32",
         "wdtype": "float32", "residual": "", "to8": False, "train": True},
        # a long prompt's rows in front of products in 8 bits, the residual
        # stream kept in float32
        {"name": "norm_to8", "kind": "norm", "n": 32768, "d": 5120, "dtype": "bfloat16",
         "wdtype": "bfloat16", "residual": "float32", "to8": True, "train": False},
        # the rows between an expert's two products brought to 8 bits
        {"name": "rows_to8", "kind": "to8", "n": 65536, "d1": 1536, "d2": 0,
         "dtype": "bfloat16"},
        # a layer's weights brought to 8 bits when a model is loaded
        {"name": "weights_to8", "kind": "to8", "n": 64, "d1": 2048, "d2": 1536,
         "dtype": "bfloat16"},
        # the experts of a few rows being answered: the weights' bytes count
        {"name": "mm_answer", "kind": "mm", "n": 32, "k": 6, "e": 64, "d1": 2048, "d2": 1408,
         "dtype": "bfloat16", "padded": False, "train": False},
        # a training batch's rows through their experts, and the gradients
        {"name": "mm_train", "kind": "mm", "n": 16384, "k": 4, "e": 64, "d1": 2048, "d2": 1536,
         "dtype": "bfloat16", "padded": False, "train": True},
        # odd widths in float16, a padded batch (rows of no expert), trained
        {"name": "mm_train_odd", "kind": "mm", "n": 10001, "k": 3, "e": 24, "d1": 602, "d2": 301,
         "dtype": "float16", "padded": True, "train": True},
        # a few rows being answered by experts kept in 8 bits
        {"name": "mm8_answer", "kind": "mm8", "n": 32, "k": 8, "e": 256, "d1": 2048, "d2": 1536,
         "dtype": "bfloat16", "padded": False},
        # a long prompt through experts kept in 8 bits
        {"name": "mm8_prompt", "kind": "mm8", "n": 32768, "k": 2, "e": 32, "d1": 4096, "d2": 2048,
         "dtype": "bfloat16", "padded": False},
        # one dense layer in 8 bits, a ragged number of rows
        {"name": "mm8_dense", "kind": "mm8", "n": 10001, "k": 1, "e": 1, "d1": 4096, "d2": 8192,
         "dtype": "bfloat16", "padded": False},
    ]


def _between(rng, lo, hi):
    """A whole number, its logarithm spread evenly over [lo, hi]."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row width: half of them any number, half whole vectors."""
    w = _between(rng, lo, hi)
    return w if rng.random() < 0.5 else max(16, w // 16 * 16)


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm", "to8", "mm", "mm", "mm", "mm8", "mm8"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    if kind == "norm":
        dtype = rng.choice([dtype, dtype, "float32"])
        d = _width(rng, 24, 16384)
        to8 = rng.random() < 0.3
        return {"kind": kind, "n": _between(rng, 1, 134000000 // d), "d": d, "dtype": dtype,
                "wdtype": rng.choice([dtype, "float32"]),
                "residual": rng.choice(["", dtype, dtype, "float32"]), "to8": to8,
                "train": not to8 and rng.random() < 0.6}
    if kind == "to8":
        if rng.random() < 0.5:
            d = _width(rng, 24, 16384)
            return {"kind": kind, "n": _between(rng, 1, 134000000 // d), "d1": d, "d2": 0,
                    "dtype": dtype}
        d1, d2 = _width(rng, 64, 8192), _width(rng, 64, 8192)
        return {"kind": kind, "n": _between(rng, 1, max(2, min(256, 200000000 // (d1 * d2)))),
                "d1": d1, "d2": d2, "dtype": dtype}
    d1, d2 = _width(rng, 32, 8192), _width(rng, 32, 8192)
    most = 200000000 if kind == "mm" else 800000000
    e = _between(rng, 1, max(2, min(256, most // (d1 * d2))))
    k = rng.randint(1, min(8, e))
    train = kind == "mm" and rng.random() < 0.5
    flops = 1.2e12 / (6 if train else 2) / (d1 * d2 * k)
    n = _between(rng, 1, max(2, min(131072 // k, int(flops), 270000000 // (max(d1, d2) * k))))
    case = {"kind": kind, "n": n, "k": k, "e": e, "d1": d1, "d2": d2, "dtype": dtype,
            "padded": rng.random() < 0.25}
    return dict(case, train=train) if kind == "mm" else case


# ---------------------------------------------------------------- inputs


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=gen).to(dtype)


def _dtype(name):
    return getattr(torch, name)


def _weights8(gen, e, d1, d2):
    """Weights as a model kept in 8 bits brings them: e4m3 values of blocks of 128 by
    128, the product's inner axis contiguous, and the blocks' scales."""
    b1, b2 = -(-d1 // _BLOCK), -(-d2 // _BLOCK)
    scale = torch.exp(0.3 * _normal(gen, e, b1, b2)) / (100.0 * math.sqrt(d1))
    data = torch.empty(e, d2, d1, dtype=torch.float8_e4m3fn, device="cuda")
    step = max(1, (1 << 27) // (d1 * d2))
    for i in range(0, e, step):
        part = data[i:i + step]
        part.copy_((100.0 * _normal(gen, *part.shape)).clamp(-_TOP, _TOP))
    return data.transpose(1, 2), scale


def _inputs(case, seed):
    """The input tensors of a case, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, n, x = case["kind"], case["n"], {}
    dt = _dtype(case["dtype"])
    if kind == "norm":
        d = case["d"]
        # a residual stream's columns are of unequal size
        col = torch.exp(0.5 * _normal(gen, d))
        x["x"] = (_normal(gen, n, d) * col).to(dt)
        x["w"] = (1.0 + 0.1 * _normal(gen, d)).to(_dtype(case["wdtype"]))
        if case["residual"]:
            x["r"] = (2.0 * _normal(gen, n, d) * col).to(_dtype(case["residual"]))
        if case["train"]:
            x["dy"] = _normal(gen, n, d, dtype=dt)
            if case["residual"]:
                x["dt"] = _normal(gen, n, d, dtype=_dtype(case["residual"]))
        return x
    d1, d2 = case["d1"], case["d2"]
    if kind == "to8":
        if d2:
            x["w"] = (_normal(gen, n, d1, d2) / math.sqrt(d1)).to(dt)
        else:
            x["x"] = (_normal(gen, n, d1) * torch.exp(0.5 * _normal(gen, d1))).to(dt)
        return x
    e, k = case["e"], case["k"]
    # experts that a bias keeps nearly balanced
    x["ids"] = torch.topk(_normal(gen, n, e) + 0.2 * _normal(gen, e), k, dim=1).indices
    if case["padded"]:  # a tenth of the batch is no row at all
        x["ids"][n - n // 10:] = -1
    x["x"] = (_normal(gen, n * k, d1) * torch.exp(0.3 * _normal(gen, d1))).to(dt)
    if kind == "mm8":
        x["w"], x["ws"] = _weights8(gen, e, d1, d2)
        return x
    x["w"] = (_normal(gen, e, d1, d2) / math.sqrt(d1)).to(dt)
    if case["train"]:
        x["dy"] = _normal(gen, n * k, d2, dtype=dt)
    return x


def _ops():
    package = os.path.join(os.getcwd(), "mojo-dgl_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import mojodgl.ops as ops

    return ops


def prepare(case, seed):
    x = _inputs(case, seed)
    x["case"] = case
    if "ids" in x:
        # the batch's layout: which entries each expert has, kept for the
        # products of a layer
        flat, e = x["ids"].reshape(-1), case["e"]
        seglen = torch.bincount(flat[flat >= 0], minlength=e)
        m, longest = int(seglen.sum()), max(1, int(seglen.max()))
        if own:
            x["plan"] = _ops().route_plan(x["ids"], e)
            if case["kind"] == "mm8":
                x["w"] = _ops().Quantized(x["w"], x["ws"])
        else:
            at = torch.arange(longest, device="cuda")
            x["live"] = at < seglen.unsqueeze(1)
            x["pad"] = (seglen.cumsum(0) - seglen).unsqueeze(1) + at
            x["pad"][~x["live"]] = 0
            x["rows"] = m
    if own and case.get("train"):
        for name in ("x", "r", "w"):
            if name in x:
                x[name].requires_grad_(True)
    return x


def run(state):
    return (_run_own if own else _run_plain)(state)


# ---------------------------------------------------------------- the package's operators


def _run_own(x):
    ops, case = _ops(), x["case"]
    kind, train = case["kind"], case.get("train", False)
    if kind == "norm":
        out = ops.rms_norm(x["x"], x["w"], x.get("r"), quantize=case["to8"])
        y, total = out if case["residual"] else (out, None)
        if case["to8"]:
            return [y.data, y.scale, total]
        if not train:
            return [y, total]
        if total is None:
            return [y.detach()] + list(torch.autograd.grad(y, (x["x"], x["w"]), x["dy"]))
        grads = torch.autograd.grad((y, total), (x["x"], x["w"], x["r"]), (x["dy"], x["dt"]))
        return [y.detach(), total.detach()] + list(grads)
    if kind == "to8":
        q = ops.quantize_blocks(x["w"]) if case["d2"] else ops.quantize_rows(x["x"])
        return [q.data, q.scale]
    if kind == "mm8":
        return [ops.scaled_mm(x["x"], x["w"], x["plan"])]
    y = ops.expert_mm(x["x"], x["w"], x["plan"])
    if not train:
        return [y]
    return [y.detach()] + list(torch.autograd.grad(y, (x["x"], x["w"]), x["dy"]))


# ---------------------------------------------------------------- the plain form


def _blocks(v, axis):
    """The axis cut into blocks of 128 (zeros fill the last), an axis more."""
    d = v.shape[axis]
    short = -d % _BLOCK
    if short:
        shape = list(v.shape)
        shape[axis] = short
        v = torch.cat([v, v.new_zeros(shape)], axis)
    return v.unflatten(axis, (-1, _BLOCK))


def _scale_of(top):
    return (top / _TOP).clamp_min(_LEAST)


def _rows8(v):
    """float32 rows as e4m3 values and the scales of their blocks of 128."""
    b = _blocks(v, 1)
    scale = _scale_of(b.abs().amax(2))
    q = (b / scale.unsqueeze(2)).to(torch.float8_e4m3fn)
    return q.flatten(1)[:, :v.shape[1]], scale


def _plain_norm(x, case):
    v, w = x["x"].float(), x["w"].float()
    t = v + x["r"].float() if case["residual"] else v
    r = torch.rsqrt((t * t).mean(1, keepdim=True) + 1e-6)
    xh = t * r
    y = xh * w
    total = t.to(x["r"].dtype) if case["residual"] else None
    if case["to8"]:
        return [*_rows8(y), total]
    out = [y.to(x["x"].dtype), total]
    if not case["train"]:
        return out
    dy = x["dy"].float()
    g = dy * w
    dx = r * (g - xh * (g * xh).mean(1, keepdim=True))
    dw = (dy * xh).sum(0).to(x["w"].dtype)
    if total is None:
        return [out[0], dx.to(x["x"].dtype), dw]
    dx = dx + x["dt"].float()
    return out + [dx.to(x["x"].dtype), dw, dx.to(x["r"].dtype)]


def _padded(rows, x):
    """(experts, longest, d) float32: each expert's rows, zeros behind them."""
    return rows.float()[x["pad"]] * x["live"].unsqueeze(2)


def _unpadded(batch, x, like):
    """The rows of the experts one after the other, zeros behind the last."""
    out = torch.zeros(like.shape[0], batch.shape[2], dtype=like.dtype, device=batch.device)
    out[:x["rows"]] = batch[x["live"]].to(like.dtype)
    return out


def _plain_mm(x, case):
    a, w = _padded(x["x"], x), x["w"].float()
    y = _unpadded(torch.bmm(a, w), x, x["x"])
    if not case["train"]:
        return [y]
    g = _padded(x["dy"], x)
    dx = torch.bmm(g, w.transpose(1, 2).contiguous())
    dw = torch.bmm(a.transpose(1, 2).contiguous(), g)
    return [y, _unpadded(dx, x, x["x"]), dw.to(x["w"].dtype)]


def _plain_mm8(x, case):
    q, scale = _rows8(x["x"].float())
    d1, d2 = case["d1"], case["d2"]
    a = q.float() * scale.repeat_interleave(_BLOCK, 1)[:, :d1]
    spread = x["ws"].repeat_interleave(_BLOCK, 1)[:, :d1].repeat_interleave(_BLOCK, 2)[..., :d2]
    w = x["w"].float() * spread
    return [_unpadded(torch.bmm(_padded(a, x), w.contiguous()), x, x["x"])]


def _run_plain(x):
    case = x["case"]
    kind = case["kind"]
    if kind == "norm":
        return _plain_norm(x, case)
    if kind == "mm":
        return _plain_mm(x, case)
    if kind == "mm8":
        return _plain_mm8(x, case)
    if not case["d2"]:
        return list(_rows8(x["x"].float()))
    b = _blocks(_blocks(x["w"].float(), 1), 3)  # (n, blocks, 128, blocks, 128)
    scale = _scale_of(b.abs().amax((2, 4)))
    q = (b / scale[:, :, None, :, None]).flatten(3).flatten(1, 2)
    q = q[:, :case["d1"], :case["d2"]].transpose(1, 2).contiguous()
    return [q.to(torch.float8_e4m3fn).transpose(1, 2), scale]


# ---------------------------------------------------------------- exact results


def _to_e4m3(v):
    """The nearest multiples of e4m3's steps, ties to even: 2^(e - 3) for values of
    [2^e, 2^(e + 1)), and no step below 2^-9."""
    e = torch.frexp(v.abs().clamp_min(2.0 ** -6)).exponent - 1
    step = torch.ldexp(torch.ones_like(v), e - 3)
    return torch.round(v / step) * step


def _exact_rows8(v):
    """e4m3 values and scales of float64 rows, block by block."""
    q, scales = torch.empty_like(v), []
    for c in range(0, v.shape[1], 128):
        part = v[:, c:c + 128]
        s = (part.abs().amax(1) / 448).clamp_min(2.0 ** -126)
        scales.append(s)
        q[:, c:c + 128] = _to_e4m3(part / s.unsqueeze(1))
    return q, torch.stack(scales, 1)


def _exact_norm(x, case):
    leaves = [x[name].double().requires_grad_(case["train"]) for name in ("x", "w", "r")
              if name in x]
    v, w = leaves[:2]
    t = v + leaves[2] if case["residual"] else v
    y = t / (t.square().mean(1, keepdim=True) + 1e-6).sqrt() * w
    total = t if case["residual"] else None
    if case["to8"]:
        return [*_exact_rows8(y), total]
    if not case["train"]:
        return [y, total]
    if total is None:
        return [y.detach()] + list(torch.autograd.grad(y, leaves, x["dy"].double()))
    grads = torch.autograd.grad((y, total), leaves, (x["dy"].double(), x["dt"].double()))
    return [y.detach(), total.detach()] + list(grads)


def _experts_of(x, case):
    """(first row, rows) of each expert."""
    flat, at, parts = x["ids"].reshape(-1), 0, []
    for e in range(case["e"]):
        m = int((flat == e).sum())
        parts.append((at, m))
        at += m
    return parts


def _exact_mm(x, case):
    a = x["x"].double()
    y = a.new_zeros(a.shape[0], case["d2"])
    train = case["train"]
    if train:
        dx, dw = torch.zeros_like(a), torch.zeros_like(x["w"], dtype=torch.float64)
    for e, (at, m) in enumerate(_experts_of(x, case)):
        if not m:
            continue
        w = x["w"][e].double()
        y[at:at + m] = a[at:at + m] @ w
        if train:
            g = x["dy"][at:at + m].double()
            dx[at:at + m] = g @ w.t().contiguous()
            dw[e] = a[at:at + m].t().contiguous() @ g
    return [y, dx, dw] if train else [y]


def _exact_mm8(x, case):
    q, scale = _exact_rows8(x["x"].double())
    d1, d2 = case["d1"], case["d2"]
    y = q.new_zeros(q.shape[0], d2)
    for e, (at, m) in enumerate(_experts_of(x, case)):
        for c in range(0, d1 if m else 0, 128):
            rows = q[at:at + m, c:c + 128] * scale[at:at + m, c // 128].unsqueeze(1)
            w = x["w"][e, c:c + 128].double().contiguous()
            col = x["ws"][e, c // 128].double().repeat_interleave(128)[:d2]
            y[at:at + m] += rows @ w * col
    return [y]


def exact(case, seed):
    x = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm":
        return _exact_norm(x, case)
    if kind == "mm":
        return _exact_mm(x, case)
    if kind == "mm8":
        return _exact_mm8(x, case)
    if not case["d2"]:
        return list(_exact_rows8(x["x"].double()))
    w = x["w"].double()
    d1, d2 = case["d1"], case["d2"]
    scale = w.new_empty(case["n"], -(-d1 // 128), -(-d2 // 128))
    for i in range(0, d1, 128):
        for j in range(0, d2, 128):
            part = w[:, i:i + 128, j:j + 128]
            s = (part.abs().amax((1, 2)) / 448).clamp_min(2.0 ** -126)
            scale[:, i // 128, j // 128] = s
            w[:, i:i + 128, j:j + 128] = _to_e4m3(part / s[:, None, None])
    return [w, scale]


# ---------------------------------------------------------------- work

_SIZE = {"float64": 8, "float32": 4, "bfloat16": 2, "float16": 2}


def work(case):
    kind, n, t = case["kind"], case["n"], _SIZE[case["dtype"]]
    train = case.get("train", False)
    if kind == "norm":
        d, tw, tr = case["d"], _SIZE[case["wdtype"]], _SIZE.get(case["residual"], 0)
        # x and the residual read, y and the sum written; backward: their
        # gradients the other way round
        row = 1 + t + 2 * tr + 4.0 / _BLOCK if case["to8"] else 2 * t + 2 * tr
        return {"bytes": n * d * row * (2 if train else 1) + d * tw * (2 if train else 1),
                "flops": n * d * (16 if train else 6)}
    d1, d2 = case["d1"], case["d2"]
    if kind == "to8":
        values, per = n * d1 * max(d2, 1), _BLOCK * _BLOCK if d2 else _BLOCK
        return {"bytes": values * (t + 1) + 4.0 * values / per, "flops": 3 * values}
    m, e = n * case["k"], case["e"]
    m = m * 0.9 if case["padded"] else m
    called = e * (1.0 - (1.0 - 1.0 / e) ** m)  # experts that any row calls, on average
    if kind == "mm8":
        return {"bytes": m * (d1 + d2) * t + called * d1 * d2, "flops": 2 * m * d1 * d2}
    # rows and weights read, the products written; backward: their gradients
    # the other way round, none of the inputs read again
    return {"bytes": (m * (d1 + d2) + called * d1 * d2) * t * (2 if train else 1),
            "flops": 2 * m * d1 * d2 * (3 if train else 1)}

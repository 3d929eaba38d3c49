"""Performance cases of the operators that training around the embeddings needs.

The norm of a sample's groups of channels with its activation (``group``), the
learned bias of an attention's scores by relative position (``bias``) and the
global norm of a model's gradients with the clipping (``clip``).  Training cases
run the forward and the backward operator, serving cases the forward alone.

A case is a dict of plain values with an ``op`` and its sizes:

``group``  ``n`` samples of ``rows`` positions (features, pixels) and ``c``
           channels (last in memory) in ``groups``; the type of the rows and of
           the parameters; the activation
``bias``   ``heads``, ``q`` queries and ``k`` keys; ``batch`` > 0: so many samples,
           whose first query stands at a position of its own; ``buckets`` of
           distances (exact up to half of them, then by logarithm up to ``far``),
           of each side or (``causal``) of the past alone, with the future
           masked; the table's and the output's type
``clip``   the gradients of a model: ``model`` "columns" (embeddings of ``rows``
           numerical features, blocks over all of them) or "text" (a table of
           ``rows`` tokens), ``blocks`` of width ``d``; the gradients' type; ``out``:
           "same" (in place, all of them in one buffer and the norm below the
           limit) or the type of the buffer that the clipped gradients of
           separate tensors go to; the kind of norm

Where ``own`` is false, ``run`` computes the same with elementary torch
operations in 32 bits, rounded once where a result is stored.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


def _group(name, n, rows, c, groups, *, dtype="bf16", params=None, activation="silu", train=True):
    return {"name": name, "op": "group", "n": n, "rows": rows, "c": c, "groups": groups, "dtype": dtype,
            "params": params or dtype, "activation": activation, "train": train}


def _bias(name, heads, q, k, *, batch=0, buckets=32, far=128, causal=False, weight="bf16", out=None, train=True):
    return {"name": name, "op": "bias", "heads": heads, "q": q, "k": k, "batch": batch, "buckets": buckets, "far": far,
            "causal": causal, "weight": weight, "out": out or weight, "train": train}


def _clip(name, model, rows, d, blocks, *, dtype="bf16", out="bf16", norm="2"):
    return {"name": name, "op": "clip", "model": model, "rows": rows, "d": d, "blocks": blocks, "dtype": dtype, "out": out,
            "norm": norm}


def listed():
    return [
        # a small tabular batch: the embeddings of 8 features
        _group("group_tiny", 256, 8, 24, 4, dtype="f32"),
        # the embeddings of 64 numerical features, 64 wide, in 32 bits
        _group("group_columns", 16384, 64, 64, 8, dtype="f32", activation="gelu"),
        # a convolutional model's training batch, 64 x 64 positions
        _group("group_image", 16, 4096, 320, 32, params="f32"),
        # the same at 256 x 256 positions
        _group("group_large", 8, 65536, 256, 32, params="f32"),
        # three samples of odd sizes, served: rows that are not multiples of 16 bytes
        _group("group_odd", 3, 1023, 250, 10, dtype="f16", activation="none", train=False),
        # one token for each of 64 requests of different lengths
        _bias("bias_decode", 32, 1, 4097, batch=64, causal=True, weight="f32", out="bf16", train=False),
        # an encoder's training step at 2048 positions
        _bias("bias_text", 16, 2048, 2048, weight="f32", out="bf16"),
        # odd lengths in 32 bits, another number of queries than of keys
        _bias("bias_odd", 12, 1023, 1301, buckets=40, far=200, weight="f32"),
        # a decoder's training step at 4096 positions
        _bias("bias_large", 16, 4096, 4096, buckets=64, far=1024, causal=True),
        # a tabular model of 24 features: 33 tensors, nothing to clip
        _clip("clip_columns", "columns", 24, 32, 4, dtype="f32", out="same"),
        # the largest gradient of a small text model, 32 bits
        _clip("clip_largest", "text", 32000, 512, 12, dtype="f32", out="f32", norm="inf"),
        # a text model in bfloat16, clipped into the optimizer's 32-bit gradients
        _clip("clip_text", "text", 50257, 1024, 24, out="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_group(rng, train):
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    if rng.random() < 0.4:      # features' embeddings
        c = rng.choice([8, 16, 24, 32, 48, 60, 64, 96, 128, 192])
        rows, most = _log(rng, 2, 300), 30_000_000
        n = max(1, min(_log(rng, 16, 65536), most // (rows * c)))
    else:                       # positions
        c = rng.choice([32, 64, 100, 128, 192, 250, 256, 320, 480, 512, 640, 960, 1024, 1280, 2048])
        rows, most = _log(rng, 16, 70000), 60_000_000
        rows = min(rows, most // c)
        n = max(1, min(_log(rng, 1, 64), most // (rows * c)))
    groups = rng.choice([g for g in (1, 2, 4, 5, 8, 10, 16, 20, 32) if c % g == 0])
    return _group("", n, rows, c, groups, dtype=dtype, params=rng.choice([dtype, "f32"]),
                  activation=rng.choice(["none", "relu", "silu", "silu", "gelu"]), train=train)


def _draw_bias(rng, train):
    heads, buckets = rng.randint(1, 40), rng.choice([8, 16, 32, 32, 40, 64, 128])
    far = buckets * rng.randint(1, 16)
    weight, out = rng.choice([("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32"), ("f16", "f16")])
    batch = 0
    if train:
        k = _log(rng, 16, 4096)
        q = k if rng.random() < 0.5 else _log(rng, 16, 4096)
    else:
        batch, q, k = rng.choice([0, _log(rng, 1, 128)]), rng.choice([1, 1, 1, 2, 5]), _log(rng, 16, 20000)
        batch = min(batch, 100_000_000 // (heads * q * k))
    heads = max(1, min(heads, 100_000_000 // (q * k)))
    return _bias("", heads, q, k, batch=batch, buckets=buckets, far=far, causal=rng.random() < 0.5 or batch > 0,
                 weight=weight, out=out, train=train)


def draw(rng):
    op = rng.choice(["group", "bias", "clip"])
    train = rng.random() < 0.75
    if op == "group":
        case = _draw_group(rng, train)
    elif op == "bias":
        case = _draw_bias(rng, train)
    else:
        dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
        out, norm = rng.choice(["same", dtype, dtype, "f32"]), rng.choice(["2", "2", "2", "inf", "1"])
        if rng.random() < 0.5:
            case = _clip("", "columns", rng.randint(2, 200), rng.choice([8, 15, 16, 24, 32, 33, 64]), rng.randint(1, 8),
                         dtype=dtype, out=out, norm=norm)
        else:
            case = _clip("", "text", _log(rng, 1000, 50000), rng.choice([128, 250, 256, 512, 640, 1000, 1024]),
                         rng.randint(2, 16), dtype=dtype, out=out, norm=norm)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEVICE, generator=gen) * scale).to(dtype)


def _prepare_group(case, gen):
    n, rows, c = case["n"], case["rows"], case["c"]
    dtype, params = DTYPES[case["dtype"]], DTYPES[case["params"]]
    # channels of different levels and sizes, as a linear layer or a convolution leaves them
    level, size = _normal(gen, c), torch.exp(_normal(gen, c, scale=0.5))
    state = {"x": (_normal(gen, n, rows, c) * size + level).to(dtype), "weight": (1 + _normal(gen, c, scale=0.2)).to(params),
             "bias": _normal(gen, c, dtype=params, scale=0.2)}
    if case["train"]:
        state["grad"] = _normal(gen, n, rows, c, dtype=dtype)
    return state


def _borders(exact, buckets, far):
    """The distances at which a side's buckets begin: 0 to ``exact``, then bucket ``exact + j`` at the first integer ``d`` with
    ``log(d / exact) / log(far / exact) >= j / (buckets - exact)``, compared in whole numbers."""
    m, found, d = buckets - exact, list(range(exact + 1)), exact
    for j in range(1, m):
        while d ** m < exact ** (m - j) * far ** j:
            d += 1
        found.append(d)
    return found


def _side(case):
    """Buckets of a side, and how many of them hold one distance."""
    side = case["buckets"] if case["causal"] else case["buckets"] // 2
    return side, side // 2


def _buckets(case):
    """The table's row for each distance key - query from -far to far."""
    side, exact = _side(case)
    far = max(case["far"], exact + 1)
    borders = torch.tensor(_borders(exact, side, far))
    past = torch.bucketize(torch.arange(far + 1), borders, right=True) - 1       # of 0, 1, ... far positions back
    future = torch.zeros(far, dtype=torch.long) if case["causal"] else side + past[1:]
    return torch.cat([past.flip(0), future]).to(torch.int32)


def _prepare_bias(case, gen):
    h, q, k, batch = case["heads"], case["q"], case["k"], case["batch"]
    state = {"weight": _normal(gen, case["buckets"], h, dtype=DTYPES[case["weight"]]), "buckets": _buckets(case).to(DEVICE),
             "starts": None, "offset": max(0, k - q)}
    if batch:
        state["starts"] = torch.randint(0, max(1, k - q + 1), (batch,), device=DEVICE, generator=gen)
    if case["train"]:
        state["grad"] = _normal(gen, h, q, k, dtype=DTYPES[case["out"]])
    return state


def _shapes(case):
    rows, d, blocks = case["rows"], case["d"], case["blocks"]
    if case["model"] == "text":
        block = [(d,), (d, d), (d, d), (d, d), (d, d), (d,), (4 * d, d), (d, 4 * d)]
        return [(rows, d), *block * blocks, (d,)]
    block = [(d,), (d,), (4 * d, rows * d), (4 * d,), (rows * d, 4 * d), (rows * d,), (1, d)]
    return [(rows, 48, d), (rows, d), (rows, d), *block * blocks, (100, rows * d), (100,)]


def _prepare_clip(case, gen):
    shapes, dtype = _shapes(case), DTYPES[case["dtype"]]
    total = sum(math.prod(s) for s in shapes)
    # about the size that gradients have: their global norm is 30, or 0.3 where nothing is to be clipped
    size = (0.3 if case["out"] == "same" else 30.0) / math.sqrt(total)
    scale = [size * (0.25 + 1.5 * i / len(shapes)) for i in range(len(shapes))]
    flat = torch.empty(total, device=DEVICE, dtype=dtype if case["out"] == "same" else DTYPES[case["out"]])
    views = [part.view(s) for part, s in zip(flat.split([math.prod(s) for s in shapes]), shapes)]
    if case["out"] == "same":
        for g, a in zip(views, scale):
            g.copy_(_normal(gen, *g.shape, scale=a))
        grads, out = views, None
    else:
        grads, out = [_normal(gen, *s, dtype=dtype, scale=a) for s, a in zip(shapes, scale)], views
    # (the sum of their sizes is sqrt(total) times as much, the largest of them a few times their size)
    limit = {"2": 1.0, "1": math.sqrt(total), "inf": 100.0 if case["out"] == "same" else size}[case["norm"]]
    return {"grads": grads, "out": out, "flat": flat, "limit": limit}


_PREPARE = {"group": _prepare_group, "bias": _prepare_bias, "clip": _prepare_clip}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"case": case, **_PREPARE[case["op"]](case, gen)}


# ---------------------------------------------------------------------------
# one pass: the framework's operators
# ---------------------------------------------------------------------------

def _package():
    import piecewiselinearembeddings_optimized_amd as package

    return package


def _ops():
    _package()
    return torch.ops.rtdl_num_embeddings_cuda


def _own_group(s, case):
    ops, act = _ops(), ACTIVATIONS[case["activation"]]
    y, stats = ops.group_norm(s["x"], s["weight"], s["bias"], case["groups"], act, EPS)
    if not case["train"]:
        return y
    return [y, *ops.group_norm_backward(s["grad"], s["x"], stats, s["weight"], s["bias"], case["groups"], act,
                                        [True, True, True])]


def _own_bias(s, case):
    ops = _ops()
    out = ops.relative_bias(s["weight"], s["buckets"], s["starts"], case["q"], case["k"], s["offset"], case["causal"],
                            DTYPES[case["out"]])
    if not case["train"]:
        return out
    return [out, ops.relative_bias_backward(s["grad"], s["buckets"], s["starts"], s["weight"].shape[0], s["offset"],
                                            case["causal"], s["weight"].dtype)]


def _own_clip(s, case):
    norm = _package().clip_gradients_(s["grads"], s["limit"], float(case["norm"]), out=s["out"])
    return [norm, s["flat"]]


# ---------------------------------------------------------------------------
# one pass: elementary operations
# ---------------------------------------------------------------------------

def _plain_activation(z, kind):
    """The activation and its derivative."""
    if kind == "relu":
        return z.clamp_min(0), (z > 0).float()
    if kind == "silu":
        sig = torch.sigmoid(z)
        return z * sig, sig * (1 + z * (1 - sig))
    if kind == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, 1.0


def _plain_group(s, case):
    n, rows, c, groups = case["n"], case["rows"], case["c"], case["groups"]
    parts = (n, rows, groups, c // groups)
    x = s["x"].float().reshape(parts)
    x = x - x.mean((1, 3), keepdim=True)
    rho = torch.rsqrt((x * x).mean((1, 3), keepdim=True) + EPS)
    xhat = x * rho
    weight, bias = s["weight"].float().reshape(parts[2:]), s["bias"].float().reshape(parts[2:])
    y, slope = _plain_activation(xhat * weight + bias, case["activation"])
    y = y.reshape(n, rows, c).to(s["x"].dtype)
    if not case["train"]:
        return y
    dz = s["grad"].float().reshape(parts) * slope
    dw, db = (dz * xhat).sum((0, 1)), dz.sum((0, 1))
    g = dz * weight
    dx = rho * (g - g.mean((1, 3), keepdim=True) - xhat * (g * xhat).mean((1, 3), keepdim=True))
    return [y, dx.reshape(n, rows, c).to(s["x"].dtype), dw.reshape(c).to(s["weight"].dtype),
            db.reshape(c).to(s["bias"].dtype)]


def _plain_bias(s, case):
    q, k, far = case["q"], case["k"], s["buckets"].shape[0] // 2
    first = torch.tensor([s["offset"]], device=DEVICE) if s["starts"] is None else s["starts"]
    at = first[:, None] + torch.arange(q, device=DEVICE)
    distance = torch.arange(k, device=DEVICE) - at[..., None]
    rows = s["buckets"][distance.clamp(-far, far) + far].long()
    out = s["weight"].t().float()[:, rows].transpose(0, 1)          # [batch, heads, q, k]
    if case["causal"]:
        out = torch.where((distance > 0)[:, None], -math.inf, out)
    out = out.to(DTYPES[case["out"]]).contiguous()
    if s["starts"] is None:
        out = out[0]
    if not case["train"]:
        return out
    g = s["grad"].float()
    if case["causal"]:
        g = torch.where(distance > 0, 0.0, g)
    # sums along the diagonals: rows in reverse, each a place further than the one before
    width = q + k
    diagonals = torch.nn.functional.pad(g.flip(1), (0, q)).reshape(-1, q * width)[:, :q * (width - 1)]
    diagonals = diagonals.reshape(-1, q, width - 1).sum(1)
    distance = torch.arange(width - 1, device=DEVICE) - (q - 1) - s["offset"]
    rows = s["buckets"][distance.clamp(-far, far) + far].long()
    own_row = (rows[:, None] == torch.arange(s["weight"].shape[0], device=DEVICE)).float()
    return [out, (diagonals[:, :, None] * own_row).sum(1).t().to(s["weight"].dtype)]


def _plain_clip(s, case):
    if case["norm"] == "inf":
        norm = torch.stack([g.abs().max() for g in s["grads"]]).float().max()
    elif case["norm"] == "1":
        norm = torch.stack([g.float().abs().sum() for g in s["grads"]]).sum()
    else:
        norm = torch.stack([(g.float() ** 2).sum() for g in s["grads"]]).sum().sqrt()
    factor = (s["limit"] / (norm + 1e-6)).clamp_max(1.0)
    if s["out"] is None:
        s["flat"].mul_(factor)
    else:
        torch.cat([(g.float() * factor).to(s["flat"].dtype).reshape(-1) for g in s["grads"]], out=s["flat"])
    return [norm, s["flat"]]


_RUN = {
    True: {"group": _own_group, "bias": _own_bias, "clip": _own_clip},
    False: {"group": _plain_group, "bias": _plain_bias, "clip": _plain_clip},
}


def run(state):
    case = state["case"]
    with torch.no_grad():
        return _RUN[bool(own)][case["op"]](state, case)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "group":
        size, param = SIZE[case["dtype"]], SIZE[case["params"]]
        values = case["n"] * case["rows"] * case["c"]
        moved, flops = 2 * values * size + 2 * case["c"] * param, 10 * values
        if case["train"]:
            # the gradient in, the rows again, their gradient out
            moved += 3 * values * size + 4 * case["c"] * param
            flops += 25 * values
        return {"bytes": moved, "flops": flops}
    if case["op"] == "bias":
        h, q, k, size = case["heads"], case["q"], case["k"], SIZE[case["out"]]
        moved = max(1, case["batch"]) * h * q * k * size + case["buckets"] * h * SIZE[case["weight"]]
        flops = 0
        if case["train"]:
            seen = q * k
            if case["causal"]:
                first = max(0, k - q)       # keys before the first query; the query itself is seen too
                seen = sum(min(k, first + i + 1) for i in range(q))
            moved += h * seen * size + case["buckets"] * h * SIZE[case["weight"]]
            flops = h * seen
        return {"bytes": moved, "flops": max(1, flops)}
    values = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": values * (SIZE[case["dtype"]] + (0 if case["out"] == "same" else SIZE[case["out"]])),
            "flops": values * (2 if case["out"] == "same" else 3)}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"group": _exact_group, "bias": _exact_bias, "clip": _exact_clip}[case["op"]](s, case)


def _exact_group(s, case):
    n, rows, c, groups = case["n"], case["rows"], case["c"], case["groups"]
    per = c // groups
    weight, bias = s["weight"].double(), s["bias"].double()
    ys, dxs = [], []
    dw, db = torch.zeros_like(weight), torch.zeros_like(bias)
    step = max(1, 40_000_000 // (rows * c))
    for a in range(0, n, step):     # samples that fit in 64 bits
        x = s["x"][a:a + step].double()
        m = x.shape[0]
        # by group: [samples, groups, values]
        lined = x.reshape(m, rows, groups, per).transpose(1, 2).reshape(m, groups, rows * per)
        var, mu = torch.var_mean(lined, 2, correction=0)
        sigma = (var + EPS).sqrt()
        spread = lambda t: t.repeat_interleave(per, 1)[:, None, :]  # noqa: E731  (a value a group to its channels)
        unit = (x - spread(mu)) / spread(sigma)
        z = unit * weight + bias
        if case["activation"] == "relu":
            y, slope = torch.where(z > 0, z, 0.0), torch.where(z > 0, 1.0, 0.0).double()
        elif case["activation"] == "silu":
            e = torch.exp(-z.abs())
            sig = torch.where(z >= 0, 1 / (1 + e), e / (1 + e))
            y, slope = z * sig, sig + z * sig * (1 - sig)
        elif case["activation"] == "gelu":
            normal = torch.special.ndtr(z)
            y, slope = z * normal, normal + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        else:
            y, slope = z, torch.ones_like(z)
        ys.append(y)
        if not case["train"]:
            continue
        dz = s["grad"][a:a + step].double() * slope
        db += dz.sum(1).sum(0)
        dw += (dz * unit).sum(1).sum(0)
        by_group = lambda t: t.sum(1).reshape(m, groups, per).sum(2) / (rows * per)  # noqa: E731
        first, second = by_group(dz * weight), by_group(dz * weight * unit)
        dxs.append((dz * weight - spread(first) - unit * spread(second)) / spread(sigma))
    return [torch.cat(ys), torch.cat(dxs), dw, db] if case["train"] else torch.cat(ys)


def _exact_bias(s, case):
    h, q, k, causal = case["heads"], case["q"], case["k"], case["causal"]
    side, direct = _side(case)
    far = max(case["far"], direct + 1)
    edges = torch.tensor(_borders(direct, side, far), device=DEVICE)
    table = s["weight"].double()
    keys = torch.arange(k, device=DEVICE)

    def bucket(position):
        """Buckets of all keys for queries at ``position``: how many of the side's buckets have begun, less one."""
        back = position[:, None] - keys
        row = (back.abs()[..., None] >= edges).sum(-1) - 1
        return torch.where((back < 0) & (not causal), side + row, row), back < 0

    outs, grad = [], torch.zeros_like(table)
    firsts = [s["offset"]] if s["starts"] is None else s["starts"].tolist()
    step = max(1, 1_000_000 // k)
    for first in firsts:
        one = torch.empty(h, q, k, dtype=torch.float64, device=DEVICE)
        for a in range(0, q, step):
            position = first + torch.arange(a, min(q, a + step), device=DEVICE)
            row, future = bucket(position)
            one[:, a:a + step] = table[row].movedim(-1, 0)
            if causal:
                one[:, a:a + step].masked_fill_(future, -math.inf)
            if case["train"]:
                g = s["grad"][:, a:a + step].double()
                if causal:
                    g = g.masked_fill(future, 0)
                for b in range(table.shape[0]):
                    grad[b] += (g * (row == b)).sum((1, 2))
        outs.append(one)
    out = outs[0] if s["starts"] is None else torch.stack(outs)
    return [out, grad] if case["train"] else out


def _exact_clip(s, case):
    wide = [g.double() for g in s["grads"]]
    if case["norm"] == "inf":
        norm = max(g.abs().max() for g in wide)
    elif case["norm"] == "1":
        norm = sum(g.abs().sum() for g in wide)
    else:
        norm = math.sqrt(sum(float((g * g).sum()) for g in wide))
    norm = torch.as_tensor(float(norm), dtype=torch.float64, device=DEVICE)
    factor = min(1.0, s["limit"] / (float(norm) + 1e-6))
    return [norm, torch.cat([(g * factor).reshape(-1) for g in wide])]

"""Performance cases of the operators around the numerical embeddings.

What a model has next to its numerical columns: tokens or categorical columns
(``lookup``), the residual trunk's norms (``norm``) and the loss of a student
that learns from a larger teacher's top logits (``distill``).  Training cases
run the forward and the backward operator, serving cases the forward alone.

A case is a dict of plain values with an ``op`` and its sizes:

``lookup``   ``n`` tokens (samples, with ``features`` > 0 categorical columns of
             one table each, 2 to ``rows`` categories), ``rows`` of the table,
             width ``d``, the table's and the output's type; ``ids``: how tokens
             are spread ("rank": log-uniform by id, as a vocabulary sorted by
             frequency; "mixed": the same frequencies over shuffled ids;
             "even": uniform)
``norm``     ``groups`` x ``rows`` rows of width ``d``; types of the residual
             stream, of the branch and of the parameters; norms after and
             before the block; the gate: "none", "shared" (one row), "group"
             (one row a group) or "row", and its activation
``distill``  ``n`` rows, ``v`` classes (the last ``padded`` of them masked with
             -inf), the teacher's ``k`` top logits, the logits' type, the
             temperature, with or without hard ``labels`` (then some rows are
             padding: no label, no teacher) and the teacher's ``tail`` mass

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
RESIDUAL_SCALE = 0.875
ALPHA = 0.75           # weight of the teacher against the labels
NORMS = {"none": 0, "rms": 1, "layer": 2}
ACTIVATIONS = {"none": 0, "sigmoid": 1, "tanh": 2}


def _lookup(name, n, rows, d, *, features=0, weight="bf16", out=None, ids="rank", train=True):
    return {"name": name, "op": "lookup", "n": n, "features": features, "rows": rows, "d": d, "weight": weight,
            "out": out or weight, "ids": ids, "train": train}


def _norm(name, groups, rows, d, *, post="rms", pre="rms", biases=False, gate="shared", activation="none",
          residual="bf16", branch="bf16", params="bf16", train=True):
    return {"name": name, "op": "norm", "groups": groups, "rows": rows, "d": d, "post": post, "pre": pre,
            "biases": biases, "gate": gate, "activation": activation, "residual": residual, "branch": branch,
            "params": params, "train": train}


def _distill(name, n, v, k, *, dtype="bf16", temperature=2.0, labels=True, tail=True, padded=0, train=True):
    return {"name": name, "op": "distill", "n": n, "v": v, "k": k, "dtype": dtype, "temperature": temperature,
            "labels": labels, "tail": tail, "padded": padded, "train": train}


def listed():
    return [
        # one generated token for each of 16 requests
        _lookup("lookup_decode", 16, 32000, 4096, train=False),
        # a tabular batch: 24 categorical columns of 2 to 5000 categories
        _lookup("lookup_columns", 8192, 5000, 32, features=24, weight="f32"),
        # a text model's training batch, a table of an odd number of rows
        _lookup("lookup_text", 16384, 50257, 1024),
        # a large vocabulary and a wide model
        _lookup("lookup_large", 65536, 131072, 2048, ids="mixed"),
        # a block's boundary for 8 single tokens
        _norm("norm_decode", 1, 8, 4096, train=False),
        # a tabular transformer: 1024 samples of 50 feature tokens, 32 bits, layer norms
        _norm("norm_columns", 1024, 50, 192, post="none", pre="layer", biases=True, residual="f32", branch="f32",
              params="f32"),
        # a text model's training batch in bfloat16
        _norm("norm_text", 1, 16384, 4096),
        # conditional model under autocast: a gate for each sample, odd sample length
        _norm("norm_adaptive", 32, 1025, 1152, post="layer", pre="layer", biases=True, gate="group",
              activation="tanh", residual="f32", params="f32"),
        # a tabular classifier of 100 classes
        _distill("distill_columns", 4096, 100, 10, dtype="f32", tail=False),
        # a few positions over a vocabulary
        _distill("distill_few", 24, 32000, 32, labels=False),
        # an odd vocabulary, labels and padding rows
        _distill("distill_text", 4096, 50257, 64),
        # a large vocabulary with masked columns at its end, temperature 1
        _distill("distill_large", 4096, 131072, 128, temperature=1.0, labels=False, padded=800),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "norm", "distill"])
    train = rng.random() < 0.75
    if op == "lookup":
        if rng.random() < 0.35:
            f, d = rng.randint(2, 60), rng.choice([8, 15, 16, 24, 32, 48, 64, 100])
            n = min(_log(rng, 64, 65536), 48_000_000 // (f * d))
            return {k: v for k, v in _lookup("", n, _log(rng, 10, 20000), d, features=f,
                                             weight=rng.choice(["f32", "f32", "bf16"]), ids=rng.choice(["rank", "even"]),
                                             train=train).items() if k != "name"}
        d = rng.choice([256, 512, 768, 1000, 1024, 1536, 2048, 2560, 4096])
        rows = min(_log(rng, 1000, 200_000), 200_000_000 // d)
        n = min(_log(rng, 256, 65536), 100_000_000 // d) if train else _log(rng, 1, 4096)
        weight, out = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16"), ("f16", "f16")])
        return {k: v for k, v in _lookup("", n, rows, d, weight=weight, out=out,
                                         ids=rng.choice(["rank", "mixed", "even"]), train=train).items() if k != "name"}
    if op == "norm":
        d = rng.choice([64, 96, 128, 192, 250, 384, 512, 768, 1000, 1024, 1152, 1536, 2048, 2560, 4096, 5120, 8192])
        n = min(_log(rng, 64, 131072), 48_000_000 // d) if train else _log(rng, 1, 8192)
        gate = rng.choice(["none", "shared", "shared", "group", "row"])
        groups = 1 if gate in ("none", "shared") else max(1, min(n, _log(rng, 2, 256)))
        residual, branch, params = rng.choice([("bf16", "bf16", "bf16"), ("bf16", "bf16", "bf16"), ("f32", "bf16", "f32"),
                                               ("f32", "f32", "f32"), ("f16", "f16", "f16")])
        kind = rng.choice(["rms", "rms", "layer"])
        return {k: v for k, v in _norm("", groups, max(1, n // groups), d, post=rng.choice([kind, kind, "none"]), pre=kind,
                                       biases=kind == "layer" and rng.random() < 0.7, gate=gate,
                                       activation=rng.choice(["none", "sigmoid", "tanh"]) if gate != "none" else "none",
                                       residual=residual, branch=branch, params=params, train=train).items()
                if k != "name"}
    if rng.random() < 0.3:
        v, n = _log(rng, 4, 2000), _log(rng, 256, 65536)
        n = min(n, 40_000_000 // v)
        k = rng.randint(2, max(2, min(20, v // 2)))
    else:
        v = _log(rng, 2000, 200_000)
        n = min(_log(rng, 8, 16384), 400_000_000 // v)
        k = rng.choice([8, 16, 20, 32, 50, 64, 100, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    if dtype == "f32":
        n = max(1, n // 2)
    return {key: val for key, val in _distill("", n, v, k, dtype=dtype, temperature=rng.choice([1.0, 2.0, 1.5, 4.0]),
                                              labels=rng.random() < 0.5, tail=rng.random() < 0.6,
                                              padded=v // 100 if rng.random() < 0.3 else 0, train=train).items()
            if key != "name"}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _cardinalities(case):
    """Categories of each column: 2 to ``rows``, spread over their logarithm."""
    f, most = case["features"], case["rows"]
    return [max(2, round(2 * (most / 2) ** (i / max(1, f - 1)))) for i in range(f)]


def _table_rows(case):
    return sum(_cardinalities(case)) if case["features"] else case["rows"]


def _normal(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEVICE, generator=gen) * scale).to(dtype)


def _spread(u, rows, ids):
    """Token ids in [0, rows) from uniform numbers."""
    t = (u * rows) if ids == "even" else torch.exp(u * torch.log(rows + 1.0)) - 1
    return torch.minimum(t.floor(), rows - 1).long()


def _prepare_lookup(case, gen):
    n, f, d = case["n"], case["features"], case["d"]
    rows = _table_rows(case)
    state = {"weight": _normal(gen, rows, d, dtype=DTYPES[case["weight"]], scale=d ** -0.5), "scale": d ** 0.5,
             "offsets": None}
    if f:
        cards = torch.tensor(_cardinalities(case), device=DEVICE)
        tokens = _spread(torch.rand(n, f, device=DEVICE, generator=gen), cards, case["ids"])
        missing = torch.rand(n, f, device=DEVICE, generator=gen) < 0.03
        state["tokens"] = torch.where(missing, -1, tokens)
        state["offsets"] = torch.cat([cards.new_zeros(1), cards.cumsum(0)])
    else:
        tokens = _spread(torch.rand(n, device=DEVICE, generator=gen), torch.tensor(rows, device=DEVICE), case["ids"])
        if case["ids"] == "mixed":
            tokens = torch.randperm(rows, device=DEVICE, generator=gen)[tokens]
        state["tokens"] = tokens
    if case["train"]:
        state["grad"] = _normal(gen, *state["tokens"].shape, d, dtype=DTYPES[case["out"]])
    return state


def _prepare_norm(case, gen):
    n, d = case["groups"] * case["rows"], case["d"]
    params, branch = DTYPES[case["params"]], DTYPES[case["branch"]]
    residual = DTYPES[case["residual"]]
    param = lambda kind: None if case[kind] == "none" else (1 + _normal(gen, d, scale=0.2)).to(params)  # noqa: E731
    bias = lambda kind: (_normal(gen, d, dtype=params, scale=0.1)  # noqa: E731
                         if case["biases"] and case[kind] != "none" else None)
    gates = {"none": None, "shared": 1, "group": case["groups"], "row": n}[case["gate"]]
    # rows of a trunk: outlying channels, and a stream larger than its branch
    channels = 1 + 4 * (torch.rand(d, device=DEVICE, generator=gen) < 0.01)
    state = {
        "residual": (_normal(gen, n, d, scale=2.0) * channels).to(residual),
        "branch": (_normal(gen, n, d) * channels + 0.1).to(branch),
        "post_weight": param("post"), "post_bias": bias("post"), "pre_weight": param("pre"), "pre_bias": bias("pre"),
        "gate": None if gates is None else _normal(gen, gates, d, dtype=params, scale=0.5),
    }
    if case["train"]:
        state["grad_stream"] = _normal(gen, n, d, dtype=residual)
        state["grad_normed"] = _normal(gen, n, d, dtype=branch)
    return state


def _prepare_distill(case, gen):
    n, v, k, t = case["n"], case["v"], case["k"], case["temperature"]
    live = v - case["padded"]
    start = torch.randint(0, live, (n, 1), device=DEVICE, generator=gen)
    step = torch.randint(1, max(2, live // k), (n, 1), device=DEVICE, generator=gen)
    ks = torch.arange(k, device=DEVICE)
    classes = (start + step * ks) % live
    teacher = 8 - 6 * (ks / k) ** 0.5 + _normal(gen, n, k, scale=0.5)
    logits = torch.randn(n, v, device=DEVICE, generator=gen)
    logits.scatter_add_(1, classes, 0.8 * teacher + _normal(gen, n, k, scale=0.5))
    logits[:, live:] = -math.inf
    state = {"logits": logits.to(DTYPES[case["dtype"]]), "teacher": teacher.sort(-1, descending=True).values,
             "teacher_lse": None, "labels": None, "grad": torch.full((n,), 1.0 / n, device=DEVICE)}
    if case["tail"]:
        top = torch.exp(teacher / t).sum(-1)
        state["teacher_lse"] = torch.log(top / (0.6 + 0.39 * torch.rand(n, device=DEVICE, generator=gen)))
    if case["labels"]:
        pick = torch.randint(0, k, (n, 1), device=DEVICE, generator=gen)
        free = torch.randint(0, live, (n,), device=DEVICE, generator=gen)
        labels = torch.where(torch.rand(n, device=DEVICE, generator=gen) < 0.8, classes.gather(1, pick)[:, 0], free)
        padding = torch.rand(n, device=DEVICE, generator=gen) < 0.06
        state["labels"] = torch.where(padding, -100, labels)
        classes = torch.where(padding[:, None], -1, classes)
    state["classes"] = classes
    return state


_PREPARE = {"lookup": _prepare_lookup, "norm": _prepare_norm, "distill": _prepare_distill}


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"case": case, **_PREPARE[case["op"]](case, gen)}


# ---------------------------------------------------------------------------
# one pass: the framework's operators
# ---------------------------------------------------------------------------

def _ops():
    import piecewiselinearembeddings_optimized_amd  # noqa: F401  (registers the operators)

    return torch.ops.rtdl_num_embeddings_cuda


def _own_lookup(s, case):
    ops = _ops()
    out = ops.lookup(s["tokens"], s["weight"], s["offsets"], s["scale"], -1, DTYPES[case["out"]])
    if not case["train"]:
        return out
    return [out, ops.lookup_backward(s["grad"], s["tokens"], s["offsets"], s["weight"].shape[0], s["scale"], -1,
                                     s["weight"].dtype)]


def _own_norm(s, case):
    ops = _ops()
    kinds = NORMS[case["post"]], NORMS[case["pre"]], ACTIVATIONS[case["activation"]]
    stream, normed, stats = ops.residual_norm(
        s["residual"], s["branch"], s["post_weight"], s["post_bias"], s["gate"], s["pre_weight"], s["pre_bias"], *kinds,
        RESIDUAL_SCALE, EPS, DTYPES[case["branch"]])
    if not case["train"]:
        return [stream, normed]
    need = [True, True] + [s[k] is not None for k in ("post_weight", "post_bias", "gate", "pre_weight", "pre_bias")]
    grads = ops.residual_norm_backward(
        s["grad_stream"], s["grad_normed"], stream, s["branch"], stats, s["post_weight"], s["post_bias"], s["gate"],
        s["pre_weight"], s["pre_bias"], *kinds, RESIDUAL_SCALE, need)
    return [stream, normed, *(g for g, wanted in zip(grads, need) if wanted)]


def _own_distill(s, case):
    ops = _ops()
    t = case["temperature"]
    loss, stats = ops.distillation_loss(s["logits"], s["teacher"], s["classes"], s["teacher_lse"], s["labels"], t, ALPHA)
    if not case["train"]:
        return loss
    return [loss, ops.distillation_loss_backward(s["grad"], s["logits"], s["teacher"], s["classes"], s["labels"], stats,
                                                 t, ALPHA)]


# ---------------------------------------------------------------------------
# one pass: elementary operations
# ---------------------------------------------------------------------------

def _plain_lookup(s, case):
    tokens, weight, d = s["tokens"], s["weight"], case["d"]
    valid = tokens >= 0
    row = tokens.clamp_min(0) if s["offsets"] is None else tokens.clamp_min(0) + s["offsets"][:-1]
    out = weight[row].float() * s["scale"]
    if case["features"]:
        out = torch.where(valid[..., None], out, 0.0)
    out = out.to(DTYPES[case["out"]])
    if not case["train"]:
        return out
    g = s["grad"].float()
    if case["features"]:
        g = torch.where(valid[..., None], g, 0.0)
    dw = torch.zeros(weight.shape, device=DEVICE).index_add_(0, row.reshape(-1), g.reshape(-1, d))
    return [out, (dw * s["scale"]).to(weight.dtype)]


def _plain_standardise(x, kind):
    """Standardised rows and the factor they were scaled with."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    rho = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * rho, rho


def _plain_affine(x, weight, bias):
    if weight is not None:
        x = x * weight.float()
    return x if bias is None else x + bias.float()


def _plain_norm_grad(g, xhat, rho, kind):
    g_mean = g.mean(-1, keepdim=True) if kind == "layer" else 0.0
    return rho * (g - g_mean - xhat * (g * xhat).mean(-1, keepdim=True))


def _plain_norm(s, case):
    groups, rows, d = case["groups"], case["rows"], case["d"]
    y = s["branch"].float()
    post, yhat, y_rho = y, None, None
    if case["post"] != "none":
        yhat, y_rho = _plain_standardise(y, case["post"])
        post = _plain_affine(yhat, s["post_weight"], s["post_bias"])
    wide = (-1, 1, d) if case["gate"] == "group" else (-1, d)
    grouped = (groups, rows, d) if case["gate"] == "group" else (-1, d)
    gated, act, slope = post, None, 1.0
    if s["gate"] is not None:
        raw = s["gate"].float()
        act = {"none": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[case["activation"]](raw)
        if case["activation"] != "none":
            slope = act * (1 - act) if case["activation"] == "sigmoid" else 1 - act * act
        gated = (post.reshape(grouped) * act.reshape(wide)).reshape(-1, d)
    stream = (RESIDUAL_SCALE * s["residual"].float() + gated).to(s["residual"].dtype)
    xhat, x_rho = _plain_standardise(stream.float(), case["pre"])
    normed = _plain_affine(xhat, s["pre_weight"], s["pre_bias"]).to(s["branch"].dtype)
    if not case["train"]:
        return [stream, normed]
    gn = s["grad_normed"].float()
    ds = s["grad_stream"].float() + _plain_norm_grad(gn * s["pre_weight"].float(), xhat, x_rho, case["pre"])
    dp, dgate = ds, None
    if act is not None:
        dp = (ds.reshape(grouped) * act.reshape(wide)).reshape(-1, d)
        by_gate = (ds * post).reshape(grouped)
        over = {"shared": 0, "group": 1}.get(case["gate"])
        dgate = (by_gate if over is None else by_gate.sum(over)).reshape(-1, d) * slope
    dy, dpw, dpb = dp, None, None
    if yhat is not None:
        dy = _plain_norm_grad(dp * s["post_weight"].float(), yhat, y_rho, case["post"])
        dpw, dpb = (dp * yhat).sum(0), dp.sum(0)
    kept = [(dpw, "post_weight"), (dpb, "post_bias"), (dgate, "gate"), ((gn * xhat).sum(0), "pre_weight"),
            (gn.sum(0), "pre_bias")]
    return [stream, normed, (RESIDUAL_SCALE * ds).to(stream.dtype), dy.to(s["branch"].dtype),
            *(g.to(s[k].dtype) for g, k in kept if s[k] is not None)]


def _plain_distill(s, case):
    n, t = case["n"], case["temperature"]
    z = s["logits"].float()
    u = z / t
    peak = u.max(-1, keepdim=True).values
    e = torch.exp(u - peak)
    total = e.sum(-1, keepdim=True)
    lse = peak + torch.log(total)
    valid = s["classes"] >= 0
    taught = valid.any(-1, keepdim=True)
    classes = s["classes"].clamp_min(0)
    tt = torch.where(valid, s["teacher"].float() / t, -math.inf)
    if s["teacher_lse"] is not None:
        t_lse = s["teacher_lse"].float()[:, None]
    else:
        t_peak = torch.where(taught, tt.max(-1, keepdim=True).values, 0.0)
        t_lse = torch.where(taught, t_peak + torch.log(torch.exp(tt - t_peak).sum(-1, keepdim=True)), 0.0)
    p = torch.exp(tt - t_lse)
    kd = torch.where(p > 0, p * (tt - t_lse - u.gather(1, classes) + lse), 0.0).sum(-1)
    mass = p.sum(-1, keepdim=True)
    inside, factor = None, mass
    if s["teacher_lse"] is not None:
        inside = torch.zeros(z.shape, dtype=torch.bool, device=DEVICE)
        inside[torch.arange(n, device=DEVICE)[:, None].expand_as(classes)[valid], classes[valid]] = True
        rest = torch.where(inside, 0.0, e).sum(-1, keepdim=True) / total
        rho = torch.where(taught, (1 - mass).clamp_min(0), 0.0)
        kd = kd + torch.where(rho > 0, rho * (torch.log(rho) - torch.log(rest)), 0.0)[:, 0]
        mass = mass + rho
        factor = mass - torch.where(rho > 0, rho / rest, 0.0)
    loss = ALPHA * t * t * kd
    if s["labels"] is not None:
        counted = s["labels"] >= 0
        label = s["labels"].clamp_min(0)[:, None]
        z_peak = z.max(-1, keepdim=True).values
        e1 = torch.exp(z - z_peak)
        total1 = e1.sum(-1, keepdim=True)
        ce = (z_peak + torch.log(total1) - z.gather(1, label))[:, 0]
        loss = loss + torch.where(counted, (1 - ALPHA) * ce, 0.0)
    if not case["train"]:
        return loss
    g = s["grad"][:, None]
    q = e / total
    dz = (ALPHA * t * g) * (q * factor if inside is None else torch.where(inside, q * mass, q * factor))
    dz.scatter_add_(1, classes, -(ALPHA * t * g) * p)
    if s["labels"] is not None:
        hard = torch.where(counted[:, None], (1 - ALPHA) * g, 0.0)
        dz = dz + hard * (e1 / total1)
        dz.scatter_add_(1, label, -hard)
    return [loss, dz.to(s["logits"].dtype)]


_RUN = {
    True: {"lookup": _own_lookup, "norm": _own_norm, "distill": _own_distill},
    False: {"lookup": _plain_lookup, "norm": _plain_norm, "distill": _plain_distill},
}


def run(state):
    case = state["case"]
    return _RUN[bool(own)][case["op"]](state, case)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _distinct(rows, tokens, ids):
    """Rows that are read at least once, about: each is drawn with its own probability."""
    if ids == "even":
        return rows * -math.expm1(-tokens / rows)
    # log-uniform: row r is drawn with probability log((r + 2) / (r + 1)) / log(rows + 1)
    return min(rows, tokens / math.log(rows + 1) * (1 + max(0.0, math.log(rows * math.log(rows + 1) / tokens))))


def work(case):
    if case["op"] == "lookup":
        w, o, d = SIZE[case["weight"]], SIZE[case["out"]], case["d"]
        tokens = case["n"] * max(1, case["features"])
        tables = _cardinalities(case) if case["features"] else [case["rows"]]
        read = sum(_distinct(r, case["n"], case["ids"]) for r in tables)
        size, flops = 8 * tokens + read * d * w + tokens * d * o, tokens * d
        if case["train"]:
            size += tokens * d * o + sum(tables) * d * w
            flops += 2 * tokens * d
        return {"bytes": size, "flops": flops}
    if case["op"] == "norm":
        n, d = case["groups"] * case["rows"], case["d"]
        r, y, p = SIZE[case["residual"]], SIZE[case["branch"]], SIZE[case["params"]]
        gates = {"none": 0, "shared": 1, "group": case["groups"], "row": n}[case["gate"]]
        vectors = sum(1 + case["biases"] for kind in ("post", "pre") if case[kind] != "none") + gates
        size, flops = n * d * (2 * r + 2 * y) + vectors * d * p, 14 * n * d
        if case["train"]:
            # gradients of both outputs in, of both inputs out; stream and branch read again
            size += n * d * (3 * r + 3 * y) + 2 * vectors * d * p
            flops += 30 * n * d
        return {"bytes": size, "flops": flops}
    n, v, k, size = case["n"], case["v"], case["k"], SIZE[case["dtype"]]
    once = n * v * size + 12 * n * k + n * 20
    return {"bytes": once + (once + n * v * size if case["train"] else 0), "flops": n * v * (10 if case["train"] else 5)}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"lookup": _exact_lookup, "norm": _exact_norm, "distill": _exact_distill}[case["op"]](s, case)


def _exact_lookup(s, case):
    d, rows = case["d"], s["weight"].shape[0]
    tokens = s["tokens"].reshape(-1)
    flat = tokens.clone()
    if case["features"]:
        flat += s["offsets"][torch.arange(tokens.numel(), device=DEVICE) % case["features"]]
    known = tokens >= 0
    table = s["weight"].double() * s["scale"]
    out = torch.zeros(tokens.numel(), d, dtype=torch.float64, device=DEVICE)
    out[known] = table[flat[known]]
    out = out.reshape(*s["tokens"].shape, d)
    if not case["train"]:
        return out
    del table
    grad = torch.zeros(rows, d, dtype=torch.float64, device=DEVICE)
    grad.index_add_(0, flat[known], s["grad"].reshape(-1, d)[known].double())
    return [out, grad * s["scale"]]


def _exact_norm(s, case):
    n, d = s["branch"].shape
    wide = {k: None if s[k] is None else s[k].double()
            for k in ("post_weight", "post_bias", "pre_weight", "pre_bias", "gate")}
    reps = 1 if s["gate"] is None else n // s["gate"].shape[0]
    spread = lambda t: t.repeat_interleave(reps, 0) if t.shape[0] != 1 else t  # noqa: E731

    def norm(x, kind, weight, bias):
        mu = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros(n, 1, dtype=torch.float64, device=DEVICE)
        sigma = ((x - mu).pow(2).mean(1, keepdim=True) + EPS).sqrt()
        unit = (x - mu) / sigma
        return unit * weight + (0 if bias is None else bias), unit, sigma

    def back(dout, unit, sigma, kind, weight):
        dunit = dout * weight
        project = unit * (dunit * unit).sum(1, keepdim=True) / d
        if kind == "layer":
            project = project + dunit.sum(1, keepdim=True) / d
        return (dunit - project) / sigma

    y = s["branch"].double()
    p, unit_y, sigma_y = y, None, None
    if case["post"] != "none":
        p, unit_y, sigma_y = norm(y, case["post"], wide["post_weight"], wide["post_bias"])
    h, dh = None, None
    if wide["gate"] is not None:
        x = wide["gate"]
        if case["activation"] == "sigmoid":
            h = 1 / (1 + (-x).exp())
            dh = h * (1 - h)
        elif case["activation"] == "tanh":
            h = x.tanh()
            dh = 1 - h.pow(2)
        else:
            h, dh = x, torch.ones_like(x)
    stream = RESIDUAL_SCALE * s["residual"].double() + (p if h is None else spread(h) * p)
    # the norm before the next block reads the stream as it is stored
    stored = stream.to(s["residual"].dtype).double()
    normed, unit_s, sigma_s = norm(stored, case["pre"], wide["pre_weight"], wide["pre_bias"])
    if not case["train"]:
        return [stream, normed]
    dn = s["grad_normed"].double()
    ds = s["grad_stream"].double() + back(dn, unit_s, sigma_s, case["pre"], wide["pre_weight"])
    dp = ds if h is None else ds * spread(h)
    dy = dp if unit_y is None else back(dp, unit_y, sigma_y, case["post"], wide["post_weight"])
    out = [stream, normed, RESIDUAL_SCALE * ds, dy]
    if unit_y is not None:
        out.append((dp * unit_y).sum(0))
        if wide["post_bias"] is not None:
            out.append(dp.sum(0))
    if h is not None:
        out.append((ds * p).reshape(-1, reps, d).sum(1) * dh)
    out.append((dn * unit_s).sum(0))
    if wide["pre_bias"] is not None:
        out.append(dn.sum(0))
    return out


def _exact_distill(s, case):
    n, v, t = case["n"], case["v"], case["temperature"]
    losses, grads = [], []
    step = max(1, 100_000_000 // v)
    for a in range(0, n, step):     # rows that fit in 64 bits
        at = slice(a, min(n, a + step))
        z, c = s["logits"][at].double(), s["classes"][at]
        m = z.shape[0]
        log_q = torch.log_softmax(z / t, 1)
        real = c >= 0
        taught = real.any(1)
        t_log = s["teacher"][at].double() / t
        t_log[~real] = -math.inf
        if case["tail"]:
            norm = s["teacher_lse"][at].double()
        else:
            norm = torch.where(taught, torch.logsumexp(t_log, 1), 0.0)
        t_log = t_log - norm[:, None]
        # the teacher's distribution over the classes, and which of them it names
        who, which = real.nonzero(as_tuple=True)
        p = torch.zeros(m, v, dtype=torch.float64, device=DEVICE)
        p.index_put_((who, c[who, which]), t_log[who, which].exp(), accumulate=True)
        kl = torch.zeros(m, dtype=torch.float64, device=DEVICE)
        prob = t_log[who, which].exp()
        kl.index_add_(0, who, prob * (t_log[who, which] - log_q[who, c[who, which]]))
        dz = log_q.exp() * taught[:, None]
        if case["tail"]:
            named = torch.zeros(m, v, dtype=torch.bool, device=DEVICE)
            named[who, c[who, which]] = True
            left = torch.where(taught, 1 - p.sum(1), 0.0)
            q_left = log_q.exp().masked_fill(named, 0).sum(1)
            kl = kl + torch.where(left > 0, left * (left / q_left).log(), 0.0)
            dz = torch.where(named, dz, dz * (1 - left / q_left)[:, None])
        dz = (dz - p) * (ALPHA * t)
        loss = ALPHA * t * t * kl
        if case["labels"]:
            label = s["labels"][at]
            kept = (label >= 0).nonzero()[:, 0]
            log_1 = torch.log_softmax(z[kept], 1)
            loss[kept] -= (1 - ALPHA) * log_1[torch.arange(len(kept), device=DEVICE), label[kept]]
            hard = log_1.exp()
            hard[torch.arange(len(kept), device=DEVICE), label[kept]] -= 1
            dz[kept] += (1 - ALPHA) * hard
        losses.append(loss)
        grads.append(dz * s["grad"][at].double()[:, None])
    return [torch.cat(losses), torch.cat(grads)] if case["train"] else torch.cat(losses)

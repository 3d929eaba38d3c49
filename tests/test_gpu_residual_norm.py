"""Residual norms (forward and backward) on the GPU against a 64-bit computation.

Tolerances.  A stored value of a 16-bit type is half a unit of that type off its
32-bit value; the 32-bit arithmetic before it is a few dozen roundings of
2^-24 on numbers of the row's size (a mean over D values adds at most D 2^-24 of
the mean's absolute value, in practice sqrt(D)).  So per element: (c 2^-24 + unit)
times the size of the terms that were added, with c = 64 for rows, and with the
terms' absolute sum for sums over rows.  The stream is stored in its type before
the norm reads it; the 64-bit computation takes the stored stream as given (its
own tests check the storing), so no rounding decides between two values.
"""

from __future__ import annotations

import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
NONE, RMS, LAYER = 0, 1, 2
EPS = 1e-5


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "HIP device required"
    import piecewiselinearembeddings_optimized_amd  # noqa: F401  (registers the ops)

    return torch.ops.rtdl_num_embeddings_cuda


def _unit_row(x, kind):
    """Standardised rows and their factor, in 64 bits."""
    if kind == NONE:
        return x, torch.ones(x.shape[0], 1, dtype=torch.float64)
    if kind == LAYER:
        x = x - x.mean(1, keepdim=True)
    rho = (x.square().mean(1, keepdim=True) + EPS).rsqrt()
    return x * rho, rho


def _back(g, unit, rho, kind):
    if kind == NONE:
        return g
    g = g - unit * (g * unit).mean(1, keepdim=True) - (g.mean(1, keepdim=True) if kind == LAYER else 0)
    return rho * g


def _gate(gate, act, n):
    if gate is None:
        return torch.ones(1, 1, dtype=torch.float64), torch.zeros(1, 1, dtype=torch.float64)
    x = gate.double()
    h = {0: x, 1: torch.sigmoid(x), 2: torch.tanh(x)}[act]
    slope = {0: torch.ones_like(x), 1: h * (1 - h), 2: 1 - h * h}[act]
    spread = lambda t: t.repeat_interleave(max(1, n // t.shape[0]), 0)  # noqa: E731
    return spread(h), spread(slope)


def _inputs(n, d, residual=F32, branch=F32, params=F32, post=RMS, pre=RMS, bias=False, gates=1, seed=0):
    gen = torch.Generator().manual_seed(seed + 31 * n + d)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    vec = lambda on, base: (base + 0.3 * r(d)).to(params) if on else None  # noqa: E731
    return {
        "residual": (2 * r(n, d)).to(residual), "branch": (r(n, d) + 0.5).to(branch),
        "post_weight": vec(post, 1.0), "post_bias": vec(post and bias, 0.0),
        "gate": r(gates, d).to(params) if gates else None,
        "pre_weight": vec(pre, 1.0), "pre_bias": vec(pre and bias, 0.0),
        "g_stream": r(n, d).to(residual), "g_normed": r(n, d).to(branch) if pre else None,
    }


NAMES = ("post_weight", "post_bias", "gate", "pre_weight", "pre_bias")


def _run(ops, x, post, pre, act, scale, need=(True,) * 7):
    dev = {k: None if v is None else v.to(DEV) for k, v in x.items()}
    params = [dev[k] for k in NAMES]
    stream, normed, stats = ops.residual_norm(dev["residual"], dev["branch"], *params, post, pre, act, scale, EPS,
                                              x["branch"].dtype)
    grads = ops.residual_norm_backward(dev["g_stream"], dev["g_normed"], stream, dev["branch"], stats, *params, post, pre,
                                       act, scale, list(need))
    return stream, normed, grads


def _close(name, got, ref, size, dtype, c=64):
    got = got.cpu().double()
    assert got.shape == ref.shape, name
    bound = c * 2.0 ** -24 * size + UNIT[dtype] * ref.abs() + (2.0 ** -24 if dtype == F16 else 1e-30)
    off = (got - ref).abs()
    assert bool((off <= bound).all()), (name, float((off / bound).max()))


def _check(ops, x, post, pre, act, scale):
    n, d = x["residual"].shape
    stream, normed, grads = _run(ops, x, post, pre, act, scale)
    w = {k: None if x[k] is None else x[k].double() for k in NAMES}
    one = lambda k: 1.0 if w[k] is None else w[k]  # noqa: E731
    zero = lambda k: 0.0 if w[k] is None else w[k]  # noqa: E731
    y = x["branch"].double()
    unit_y, rho_y = _unit_row(y, post)
    p = unit_y * one("post_weight") + zero("post_bias")
    h, slope = _gate(x["gate"], act, n)
    ref = scale * x["residual"].double() + h * p
    size = ((scale * x["residual"].double()).abs() + (h * p).abs()
            + (h * one("post_weight")).abs() * ((y * rho_y).abs() + (y * rho_y).abs().mean(1, keepdim=True) * (post == LAYER)))
    _close("stream", stream, ref, size, x["residual"].dtype)

    s = stream.cpu().double()           # as stored
    unit_s, rho_s = _unit_row(s, pre)
    ds = x["g_stream"].double()
    ds_size = ds.abs()
    row = lambda t: t.abs().mean(1, keepdim=True)  # noqa: E731
    # (a layer norm's mean is a sum of the row's values: its error does not shrink with an element)
    mean_size = lambda t, kind: row(t) if kind == LAYER else 0.0  # noqa: E731
    if pre:
        unit_size = unit_s.abs() + (s * rho_s).abs() + mean_size(s * rho_s, pre)
        n_size = unit_size * abs(one("pre_weight")) + abs(zero("pre_bias"))
        _close("normed", normed, unit_s * one("pre_weight") + zero("pre_bias"), n_size, x["branch"].dtype)
        gn = x["g_normed"].double()
        gw = gn * one("pre_weight")
        ds = ds + _back(gw, unit_s, rho_s, pre)
        ds_size = ds_size + rho_s * (gw.abs() + row(gw) + unit_size * (gw.abs() * unit_size).mean(1, keepdim=True))
    dp = ds * h
    dp_size = ds_size * h.abs()
    _close("d residual", grads[0], scale * ds, scale * ds_size, x["residual"].dtype)
    y_size = unit_y.abs() + (y * rho_y).abs() + mean_size(y * rho_y, post) if post else y.abs()
    p_size = y_size * abs(one("post_weight")) + abs(zero("post_bias"))
    if post:
        dw = dp * one("post_weight")
        dw_size = dp_size * abs(one("post_weight"))
        dy = _back(dw, unit_y, rho_y, post)
        dy_size = rho_y * (dw_size + row(dw_size) + y_size * (dw_size * y_size).mean(1, keepdim=True))
    else:
        dy, dy_size = dp, dp_size
    _close("d branch", grads[1], dy, dy_size, x["branch"].dtype)
    sums = {"post_weight": (dp * unit_y, dp_size * y_size), "post_bias": (dp, dp_size)}
    if pre:
        sums |= {"pre_weight": (gn * unit_s, gn.abs() * unit_size), "pre_bias": (gn, gn.abs())}
    for i, k in enumerate(NAMES):
        if w[k] is None:
            assert grads[2 + i].numel() == 0
        elif k == "gate":
            g = w[k].shape[0]
            fold = lambda t: t.expand(n, d).reshape(g, n // g, d).sum(1)  # noqa: E731
            _close("d gate", grads[4], fold(ds * p * slope), fold((ds_size * p_size + (ds * p).abs()) * slope.abs()
                                                                 + (ds * p).abs() * 2.0 ** -3 * (act != 0)),
                   x[k].dtype)
        else:
            _close("d " + k, grads[2 + i], sums[k][0].sum(0), sums[k][1].sum(0), x[k].dtype)


TYPES = [(F32, F32, F32), (BF16, BF16, BF16), (F16, F16, F16), (F32, BF16, F32), (F32, F16, F16), (BF16, BF16, F32)]


def _ids(v):
    return "-".join(str(t)[6:] for t in v)


@pytest.mark.parametrize("types", TYPES, ids=_ids)
@pytest.mark.parametrize("n,d", [(1, 1), (1, 8), (3, 7), (5, 64), (70, 65), (9, 128), (33, 200), (4, 256), (130, 264),
                                 (17, 512), (6, 520), (3, 1000), (2, 1001), (5, 1152), (3, 2048), (2, 4099), (3, 4096),
                                 (2, 5120), (2, 8191), (1, 8192)])
def test_widths(ops, n, d, types):
    _check(ops, _inputs(n, d, *types, post=LAYER, pre=RMS, bias=True), LAYER, RMS, 0, 0.75)


@pytest.mark.parametrize("act", [0, 1, 2], ids=["identity", "sigmoid", "tanh"])
@pytest.mark.parametrize("post,pre", list(itertools.product([NONE, RMS, LAYER], repeat=2)))
@pytest.mark.parametrize("bias", [False, True])
def test_kinds(ops, post, pre, act, bias):
    _check(ops, _inputs(45, 96, post=post, pre=pre, bias=bias), post, pre, act, 1.0)
    _check(ops, _inputs(45, 96, BF16, BF16, BF16, post=post, pre=pre, bias=bias, gates=0), post, pre, act, 0.5)


@pytest.mark.parametrize("types", TYPES[:4], ids=_ids)
@pytest.mark.parametrize("gates,n,d", [(1, 1, 32), (12, 12, 40), (1, 500, 72), (3, 60, 24), (7, 7 * 131, 16), (2, 8000, 48),
                                       (50, 200, 1100), (2, 600, 2056), (300, 600, 9), (1, 3000, 33), (5, 5 * 1999, 64)])
def test_gates(ops, gates, n, d, types):
    _check(ops, _inputs(n, d, *types, gates=gates), RMS, LAYER, 2, 0.9)


@pytest.mark.parametrize("n,d", [(30_000, 24), (5000, 512), (3001, 1024)])
def test_many_rows(ops, n, d):
    _check(ops, _inputs(n, d, F32, BF16, F32, bias=True, post=LAYER, pre=LAYER), LAYER, LAYER, 1, 1.0)


@pytest.mark.parametrize("types", [(F32, F32, F32), (BF16, BF16, BF16), (F32, BF16, F32)], ids=_ids)
@pytest.mark.parametrize("n,d,gates", [(1100, 4104, 1), (1099, 4100, 7), (1100, 5120, 1), (1100, 5120, 5), (1033, 6001, 0),
                                       (1100, 6144, 1), (1100, 6152, 1), (1100, 6152, 10), (1099, 8191, 1), (1100, 8192, 1),
                                       (1100, 8192, 11), (600, 8192, 600)])
def test_wide_rows_in_turn(ops, n, d, gates, types):
    """Rows of 768 and 1024 threads, several to a workgroup: the next row's loads, the
    joins' two buffers and the parameters' sums go from row to row."""
    _check(ops, _inputs(n, d, *types, bias=True, post=LAYER, pre=LAYER, gates=gates), LAYER, LAYER, 2 if gates else 0, 0.75)
    _check(ops, _inputs(n, d, *types, post=RMS, pre=RMS, gates=gates), RMS, RMS, 0, 1.0)


def test_without_weights(ops):
    x = _inputs(40, 100, gates=0)
    x["post_weight"] = x["pre_weight"] = None
    _check(ops, x, RMS, LAYER, 0, 1.0)


def test_wanted_gradients_only(ops):
    x = _inputs(20, 48, bias=True, gates=4)
    every = _run(ops, x, RMS, LAYER, 1, 0.5)[2]
    for i in range(7):
        some = _run(ops, x, RMS, LAYER, 1, 0.5, [k == i for k in range(7)])[2]
        assert torch.equal(some[i], every[i])
        assert all(t.numel() == 0 for k, t in enumerate(some) if k != i)


def test_missing_output_gradients(ops):
    """A gradient that is not given is a gradient of zeros."""
    x = _inputs(20, 48, gates=4)
    for gone in ("g_stream", "g_normed"):
        zeros = dict(x, **{gone: torch.zeros_like(x[gone])})
        for a, b in zip(_run(ops, dict(x, **{gone: None}), RMS, LAYER, 1, 0.5)[2], _run(ops, zeros, RMS, LAYER, 1, 0.5)[2]):
            torch.testing.assert_close(a, b, rtol=0, atol=0)


@pytest.mark.parametrize("kind", [RMS, LAYER])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_before_a_block_only(ops, kind, dtype):
    x = _inputs(50, 104, dtype, dtype, dtype, post=NONE, pre=kind, bias=True, gates=0)
    r, w, b = (x[k].to(DEV) for k in ("residual", "pre_weight", "pre_bias"))
    stream, normed, stats = ops.residual_norm(r, None, None, None, None, w, b, 0, kind, 0, 1.0, EPS, dtype)
    assert stream.numel() == 0
    unit, rho = _unit_row(x["residual"].double(), kind)
    ref = unit * x["pre_weight"].double() + x["pre_bias"].double()
    size = unit.abs() * 2 + 2
    _close("normed", normed, ref, size, dtype)
    g = x["g_normed"].to(DEV)
    grads = ops.residual_norm_backward(None, g, r, None, stats, None, None, None, w, b, 0, kind, 0, 1.0,
                                       [True, False, False, False, False, True, True])
    gw = x["g_normed"].double() * x["pre_weight"].double()
    _close("d residual", grads[0], _back(gw, unit, rho, kind),
           rho * (gw.abs() + 2 * gw.abs().mean(1, keepdim=True) + unit.abs() * (gw * unit).abs().mean(1, keepdim=True) + 1), dtype)
    _close("d weight", grads[5], (x["g_normed"].double() * unit).sum(0),
           (x["g_normed"].double().abs() * (unit.abs() + 1)).sum(0), dtype)


def test_rows_of_equal_and_large_values(ops):
    """A row without spread, one far from zero and one of zeros."""
    x = _inputs(6, 256, bias=True, post=LAYER, pre=LAYER, gates=0)
    x["branch"][0] = 3.0
    x["branch"][1] = 0.0
    x["residual"][2] = 1000 + torch.randn(256, generator=torch.Generator().manual_seed(1))
    x["branch"][3] *= 1e-6
    x["branch"][4] *= 1e6
    _check(ops, x, LAYER, LAYER, 0, 1.0)


def test_non_finite_rows_stay_alone(ops):
    x = _inputs(64, 40)
    want = _run(ops, x, RMS, LAYER, 0, 1.0)
    x["branch"][5, 3] = float("nan")
    x["residual"][9, 0] = float("inf")
    got = _run(ops, x, RMS, LAYER, 0, 1.0)
    rows = [i for i in range(64) if i not in (5, 9)]
    for a, b in zip((*got[:2], *got[2][:2]), (*want[:2], *want[2][:2])):
        assert torch.equal(a[rows], b[rows])
        assert torch.isnan(a[5]).any() and not torch.isfinite(a[9]).all()


@pytest.mark.parametrize("d", [64, 1024])
def test_unaligned_rows(ops, d):
    """Rows of whole vectors at addresses that are not aligned for them."""
    x = _inputs(30, d, BF16, BF16, BF16)
    want = _run(ops, x, RMS, RMS, 0, 1.0)

    def shift(t):
        if t is None:
            return None
        base = torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)
        base[1:] = t.to(DEV).reshape(-1)
        return base[1:].view(t.shape)

    dev = {k: shift(v) for k, v in x.items()}
    params = [dev[k] for k in NAMES]
    stream, normed, stats = ops.residual_norm(dev["residual"], dev["branch"], *params, RMS, RMS, 0, 1.0, EPS, BF16)
    grads = ops.residual_norm_backward(dev["g_stream"], dev["g_normed"], stream, dev["branch"], stats, *params, RMS, RMS, 0,
                                       1.0, [True] * 7)
    for a, b in zip((stream, normed, *grads), (*want[:2], *want[2])):
        torch.testing.assert_close(a, b, rtol=2e-2, atol=2e-2)


def test_unaligned_rows_with_gates_of_groups(ops):
    """Their workspace is asked for before the addresses are known."""
    x = _inputs(2570, 1152, BF16, BF16, BF16, gates=257)
    x["post_weight"] = x["pre_weight"] = None
    want = _run(ops, x, RMS, RMS, 0, 1.0)
    dev = {k: None if v is None else v.to(DEV) for k, v in x.items()}
    for k in ("residual", "branch", "g_stream", "g_normed"):
        base = torch.zeros(dev[k].numel() + 1, dtype=BF16, device=DEV)
        base[1:] = dev[k].reshape(-1)
        dev[k] = base[1:].view(dev[k].shape)
    params = [dev[k] for k in NAMES]
    stream, normed, stats = ops.residual_norm(dev["residual"], dev["branch"], *params, RMS, RMS, 0, 1.0, EPS, BF16)
    grads = ops.residual_norm_backward(dev["g_stream"], dev["g_normed"], stream, dev["branch"], stats, *params, RMS, RMS, 0,
                                       1.0, [True] * 7)
    for a, b in zip((stream, normed, *grads), (*want[:2], *want[2])):
        torch.testing.assert_close(a, b, rtol=2e-2, atol=2e-2)


def test_empty(ops):
    x = _inputs(0, 32, gates=3, bias=True)
    stream, normed, grads = _run(ops, x, RMS, LAYER, 0, 1.0)
    assert stream.shape == normed.shape == (0, 32) and grads[4].shape == (3, 32)
    assert all(not bool(g.any()) for g in grads)


def test_empty_with_many_gate_rows(ops):
    """The gradients of more gate rows than one launch joins are cleared."""
    g, d = 40_000, 8192
    none = torch.zeros(0, d, dtype=BF16, device=DEV)
    gate = torch.ones(g, d, dtype=BF16, device=DEV)
    torch.ones(g, d, dtype=BF16, device=DEV)            # (the memory that the gradient gets is not clear)
    stats = torch.zeros(0, 4, device=DEV)
    grads = ops.residual_norm_backward(none, none, none, none, stats, None, None, gate, None, None, RMS, RMS, 0, 1.0, [True] * 7)
    assert grads[4].shape == (g, d) and not bool(grads[4].any())


def test_same_bits_every_time(ops):
    x = _inputs(7001, 136, BF16, BF16, BF16, gates=7, bias=True)
    x["residual"] = x["residual"][:7000]
    x = {k: v[:7000] if v is not None and v.shape[0] == 7001 else v for k, v in x.items()}
    a, b = _run(ops, x, RMS, LAYER, 0, 1.0), _run(ops, x, RMS, LAYER, 0, 1.0)
    for u, v in zip((*a[:2], *a[2]), (*b[:2], *b[2])):
        assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))


def test_other_stream_and_graph(ops):
    x = _inputs(900, 200, gates=9)
    want = _run(ops, x, RMS, LAYER, 1, 0.5)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _run(ops, x, RMS, LAYER, 1, 0.5)
    s.synchronize()
    flat = lambda r: (*r[:2], *r[2])  # noqa: E731
    assert all(torch.equal(a, b) for a, b in zip(flat(got), flat(want)))

    dev = {k: None if v is None else v.to(DEV) for k, v in x.items()}
    params = [dev[k] for k in NAMES]

    def both():
        stream, normed, stats = ops.residual_norm(dev["residual"], dev["branch"], *params, RMS, LAYER, 1, 0.5, EPS, F32)
        return (stream, normed, *ops.residual_norm_backward(dev["g_stream"], dev["g_normed"], stream, dev["branch"], stats,
                                                            *params, RMS, LAYER, 1, 0.5, [True] * 7))

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for k in range(3):
        dev["branch"].mul_(0.5 + k)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, both())), k


@pytest.mark.parametrize("gate", ["none", "learned", "row", "sample", "channel"])
def test_module_gradients(ops, gate):
    """Module autograd against the CPU module's (plain operations), and against differences."""
    from piecewiselinearembeddings_optimized_amd import CudaResidualNorm

    torch.manual_seed(1)
    m = CudaResidualNorm(24, post_norm="layer", pre_norm="rms", bias=True, gate="learned" if gate == "learned" else None,
                         gate_activation="tanh", residual_scale=0.7)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.3 * torch.randn_like(p))
    res, br = torch.randn(6, 5, 24, requires_grad=True), torch.randn(6, 5, 24, requires_grad=True)
    g = {"row": (6, 5, 24), "sample": (6, 1, 24), "channel": (24,)}.get(gate)
    g = None if g is None else torch.randn(g, requires_grad=True)
    up = torch.randn(2, 6, 5, 24)
    leaves = [t for t in (res, br, g) if t is not None]

    def value(mod, tensors, u, double=False):
        s, n = mod(*tensors)
        f = (lambda t: t.double()) if double else (lambda t: t)
        return (f(s) * u[0]).sum() + (f(n) * u[1]).sum()

    want = torch.autograd.grad(value(m, leaves, up), [*leaves, *m.parameters()])
    md = CudaResidualNorm(24, post_norm="layer", pre_norm="rms", bias=True, gate="learned" if gate == "learned" else None,
                          gate_activation="tanh", residual_scale=0.7)
    md.load_state_dict(m.state_dict())
    md = md.to(DEV)
    dev = [t.detach().to(DEV).requires_grad_() for t in leaves]
    every = [*dev, *md.parameters()]
    got = torch.autograd.grad(value(md, dev, up.to(DEV)), every)
    for a, b in zip(got, want):
        torch.testing.assert_close(a.cpu(), b, rtol=1e-4, atol=1e-4)
    with torch.no_grad():
        step = [torch.randn_like(t) for t in every]
        h = 1e-2
        ends = []
        for sign in (h, -2 * h):
            for t, s in zip(every, step):
                t.add_(s, alpha=sign)
            ends.append(float(value(md, dev, up.to(DEV), True)))
    slope = (ends[0] - ends[1]) / (2 * h)
    along = sum(float((a.double() * s).sum()) for a, s in zip(got, step))
    # (the second difference's error is h^2 times third derivatives; 32-bit values over 2 h add about 1e-3)
    assert abs(slope - along) < 0.02 * max(1.0, sum(float((a * s).abs().sum()) for a, s in zip(got, step)) ** 0.5 * 5)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda d: str(d)[6:])
def test_gate_of_another_layout_and_dtype(ops, dtype):
    """A gate as a model makes it: a part of a wider tensor, in the autocast dtype."""
    from piecewiselinearembeddings_optimized_amd import CudaResidualNorm

    gen = torch.Generator().manual_seed(2)
    m = CudaResidualNorm(24, post_norm="rms", pre_norm="layer", gate_activation="sigmoid")
    res, br = torch.randn(6, 5, 24, generator=gen), torch.randn(6, 5, 24, generator=gen)
    wide = torch.randn(6, 1, 72, generator=gen).to(dtype)
    up = torch.randn(2, 6, 5, 24, generator=gen)

    def grads(m, dev):
        w = wide.to(dev).requires_grad_()
        s, n = m(res.to(dev), br.to(dev), w.chunk(3, -1)[1])
        return s, n, torch.autograd.grad((s * up[0].to(dev)).sum() + (n * up[1].to(dev)).sum(), w)[0]

    want = grads(m, "cpu")
    got = grads(m.to(DEV), DEV)
    assert got[2].dtype == dtype
    for a, b, tol in zip(got, want, (1e-5, 1e-5, 1e-4 if dtype == F32 else 2e-2)):
        torch.testing.assert_close(a.cpu(), b, rtol=tol, atol=tol)


def test_stream_used_twice(ops):
    """Both outputs and the residual's reuse: gradients add up as in plain autograd."""
    from piecewiselinearembeddings_optimized_amd import CudaResidualNorm

    a, b = CudaResidualNorm(16, pre_norm="rms"), CudaResidualNorm(16, post_norm="rms", pre_norm=None)
    x = torch.randn(10, 16, requires_grad=True)

    def run(a, b, x):
        s, n = a(x)
        s, n = a(s, n * 2)
        s, n = b(s, n.tanh())
        return (s * n).sum()

    want = torch.autograd.grad(run(a, b, x), [x, a.pre_weight, b.post_weight])
    a, b, xd = a.to(DEV), b.to(DEV), x.detach().to(DEV).requires_grad_()
    for g, w in zip(torch.autograd.grad(run(a, b, xd), [xd, a.pre_weight, b.post_weight]), want):
        torch.testing.assert_close(g.cpu(), w, rtol=1e-4, atol=1e-4)


def test_opcheck(ops):
    x = {k: None if v is None else v.to(DEV).requires_grad_() for k, v in _inputs(6, 16, bias=True, gates=2).items()}
    params = [x[k] for k in NAMES]
    torch.library.opcheck(ops.residual_norm.default, (x["residual"], x["branch"], *params, 1, 2, 1, 0.5, EPS, F32))
    torch.library.opcheck(ops.residual_norm.default,
                          (x["residual"], None, None, None, None, params[3], params[4], 0, 2, 0, 1.0, EPS, F32))


def test_compiled(ops):
    from piecewiselinearembeddings_optimized_amd import CudaResidualNorm

    m = CudaResidualNorm(32, post_norm="rms", pre_norm="layer", gate="learned").to(DEV)
    r, b = torch.randn(9, 32, device=DEV), torch.randn(9, 32, device=DEV, requires_grad=True)
    f = lambda r, b: sum(t.square().sum() for t in m(r, b))  # noqa: E731
    got = torch.autograd.grad(torch.compile(f, fullgraph=True)(r, b), [b, *m.parameters()])
    for a, w in zip(got, torch.autograd.grad(f(r, b), [b, *m.parameters()])):
        torch.testing.assert_close(a, w)


def test_refusals(ops):
    r, b, w = torch.randn(4, 8, device=DEV), torch.randn(4, 8, device=DEV), torch.ones(8, device=DEV)

    def call(residual=r, branch=b, post=w, post_bias=None, gate=None, pre=w, kinds=(1, 1, 0), scale=1.0, dtype=F32):
        return ops.residual_norm(residual, branch, post, post_bias, gate, pre, None, *kinds, scale, EPS, dtype)

    for match, kw in {
        "branch must have the shape": {"branch": b[:2]},
        "branch must be contiguous": {"branch": torch.randn(8, 4, device=DEV).T},
        "normed_dtype must be": {"dtype": BF16},
        "float32 or of the branch's dtype": {"residual": r.bfloat16()},
        "must be 0 \\(none\\)": {"kinds": (3, 1, 0)},
        "gate_activation must be": {"kinds": (1, 1, 5)},
        "need a post norm": {"kinds": (0, 1, 0)},
        "need a pre norm": {"kinds": (1, 0, 0)},
        "must have shape \\[D\\]": {"post": w[:4]},
        "one dtype": {"pre": w.bfloat16()},
        "must divide": {"gate": torch.ones(3, 8, device=DEV)},
        "must have shape \\[G, D\\]": {"gate": w},
        "without a branch": {"branch": None},
        "at most 8192": {"residual": torch.zeros(1, 8193, device=DEV), "branch": torch.zeros(1, 8193, device=DEV)},
        "same CUDA device": {"post": w.cpu()},
    }.items():
        with pytest.raises(RuntimeError, match=match):
            call(**kw)


def test_c_abi(ops):
    """The ctypes binding gives the operators' bits, and refuses a small workspace."""
    from piecewiselinearembeddings_optimized_amd import capi

    x = _inputs(300, 88, F32, BF16, F32, gates=3, bias=True)
    want = _run(ops, x, RMS, LAYER, 1, 0.5)
    dev = {k: v.to(DEV) for k, v in x.items()}
    d = capi.norm(F32, BF16, RMS, LAYER, **{k: dev[k] for k in NAMES}, gate_activation=1, residual_scale=0.5, eps=EPS)
    stream, normed = torch.empty_like(dev["residual"]), torch.empty_like(dev["branch"])
    stats = torch.empty(300, 4, device=DEV)
    capi.residual_norm(dev["residual"], dev["branch"], d, stream, normed, stats)
    grads = {k: torch.empty_like(dev[k]) for k in ("residual", "branch", *NAMES)}
    capi.residual_norm_backward(dev["g_stream"], dev["g_normed"], stream, dev["branch"], stats, d, grads)
    for a, b in zip((stream, normed, *grads.values()), (*want[:2], *want[2])):
        assert torch.equal(a, b)
    with pytest.raises(capi.PleError, match="workspace"):
        capi.residual_norm_backward(dev["g_stream"], dev["g_normed"], stream, dev["branch"], stats, d, grads,
                                    workspace=torch.empty(64, dtype=torch.uint8, device=DEV))

"""Group norm with its activation (forward and backward) on the GPU against a 64-bit
computation.

Tolerances.  With e = 64 * 2^-24 (a few dozen roundings of 32-bit numbers, in sums
that are trees): a standardised value is off by e times the size of what it is made
of, rho (|x| + mean |x|), and by its factor's error, which is the mean of those
times |xh|; z and y follow with |w| (no activation's slope exceeds 1.2), and the
slope of silu and gelu by at most that much again.  A relu's slope is unknown where
z is that close to 0.  Sums add their terms' errors.  A stored value of a 16-bit
type is half a unit of that type off its 32-bit value.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 1e-37, BF16: 1e-37, F16: 2.0 ** -25}
E = 64 * 2.0 ** -24
NONE, RELU, SILU, GELU = range(4)
EPS = 1e-5


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "HIP device required"
    import piecewiselinearembeddings_optimized_amd  # noqa: F401  (registers the ops)

    return torch.ops.rtdl_num_embeddings_cuda


def _activation(z, act):
    if act == RELU:
        return z.clamp_min(0), (z > 0).double()
    if act == SILU:
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if act == GELU:
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def _inputs(n, s, c, dtype=F32, params=F32, seed=0, level=1.0):
    gen = torch.Generator().manual_seed(seed + 31 * n + 7 * s + c)
    r = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
    return {"x": (r(n, s, c) * (0.5 + r(c).abs()) + level * r(c)).to(dtype), "g": r(n, s, c).to(dtype),
            "weight": None if params is None else (1 + 0.3 * r(c)).to(params),
            "bias": None if params is None else (0.3 * r(c)).to(params)}


def _reference(x, groups, act):
    """Values and their errors, in 64 bits: (y, dx, dw, db) and a bound for each."""
    n, s, c = x["x"].shape
    p = c // groups
    v = x["x"].double()
    mean = lambda t: (t.reshape(n, s, groups, p).mean((1, 3), keepdim=True).expand(n, s, groups, p)  # noqa: E731
                      .reshape(n, s, c))
    w = torch.ones(c).double() if x["weight"] is None else x["weight"].double()
    b = torch.zeros(c).double() if x["bias"] is None else x["bias"].double()
    d = v - mean(v)
    rho = (mean(d * d) + EPS).rsqrt()
    xh = d * rho
    xh_err = E * rho * (v.abs() + mean(v.abs()))
    xh_err = xh_err + xh.abs() * (mean(xh_err * xh.abs()) + E)
    z = xh * w + b
    z_err = xh_err * w.abs() + E * (xh.abs() * w.abs() + b.abs())
    y, slope = _activation(z, act)
    y_err = 1.2 * z_err + E * y.abs()
    dy = x["g"].double()
    dz = dy * slope
    if act == RELU:
        dz_err = dy.abs() * (z.abs() <= z_err)
    else:
        dz_err = dy.abs() * (z_err + E) if act != NONE else torch.zeros_like(dz)
    dz_err = dz_err + E * dz.abs()
    g, g_err = dz * w, dz_err * w.abs()
    m1, m2 = mean(g), mean(g * xh)
    dx = rho * (g - m1 - xh * m2)
    m2_err = mean(g_err * xh.abs() + g.abs() * xh_err + E * (g * xh).abs())
    dx_err = rho * (g_err + E * (g.abs() + mean(g.abs())) + mean(g_err) + xh_err * mean((g * xh).abs()) + xh.abs() * m2_err)
    dx_err = dx_err + dx.abs() * (E + mean(xh_err * xh.abs()))
    dw_err = (dz_err * xh.abs() + dz.abs() * xh_err + E * (dz * xh).abs()).sum((0, 1))
    return ([y, dx, (dz * xh).sum((0, 1)), dz.sum((0, 1))],
            [y_err, dx_err, dw_err, (dz_err + E * dz.abs()).sum((0, 1))])


def _run(ops, x, groups, act, need=(True,) * 3):
    dev = {k: None if t is None else t.to(DEV) for k, t in x.items()}
    y, stats = ops.group_norm(dev["x"], dev["weight"], dev["bias"], groups, act, EPS)
    return [y, *ops.group_norm_backward(dev["g"], dev["x"], stats, dev["weight"], dev["bias"], groups, act, list(need))], stats


def _check(ops, x, groups, act):
    got, stats = _run(ops, x, groups, act)
    ref, err = _reference(x, groups, act)
    types = [x["x"].dtype] * 2 + [F32 if x["weight"] is None else x["weight"].dtype] * 2
    for name, a, r, e, t in zip(("y", "dx", "dw", "db"), got, ref, err, types):
        if x["weight"] is None and name in ("dw", "db"):
            assert a.numel() == 0
            continue
        a = a.cpu()
        assert a.dtype == t and a.shape == r.shape, name
        bound = e + UNIT[t] * (r.abs() + e) + TINY[t]
        off = (a.double() - r).abs()
        assert bool((off <= bound).all()), (name, float((off / bound).max()))
    assert stats.shape == (x["x"].shape[0], groups, 2) and bool(torch.isfinite(stats).all())


TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32), (F32, BF16)]


def _ids(v):
    return "-".join(str(t)[6:] for t in v)


# rows, channels, groups: one value, one row, one channel a group, groups of whole and of
# broken vectors, rows that are multiples of 16, 4 and 2 bytes, several samples a wave,
# slabs, one group, rows wider than a workgroup, samples too large to be held
SIZES = [(1, 1, 1, 1), (3, 1, 8, 8), (2, 5, 6, 3), (9, 8, 24, 4), (5, 8, 24, 24), (70, 2, 8, 2), (33, 3, 16, 1), (4, 7, 250, 10),
         (3, 33, 7, 7), (3, 40, 9, 3), (2, 64, 64, 8), (2, 130, 60, 5), (2, 100, 320, 32), (1, 1023, 250, 10), (1, 1, 4096, 2),
         (2, 3, 9000, 3), (1, 2, 20000, 1), (2, 4096, 40, 4), (1, 5000, 64, 64), (2, 900, 512, 32), (1, 4097, 130, 13),
         (3, 300, 1280, 32), (2, 2100, 77, 7), (1, 20011, 24, 3)]


@pytest.mark.parametrize("types", TYPES, ids=_ids)
@pytest.mark.parametrize("n,s,c,groups", SIZES)
def test_sizes(ops, n, s, c, groups, types):
    _check(ops, _inputs(n, s, c, *types), groups, SILU)


@pytest.mark.parametrize("act", [NONE, RELU, SILU, GELU], ids=["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("n,s,c,groups", [(20, 12, 48, 6), (3, 700, 96, 8), (2, 6000, 50, 5)])
def test_activations(ops, n, s, c, groups, dtype, act):
    _check(ops, _inputs(n, s, c, dtype, F32), groups, act)
    _check(ops, _inputs(n, s, c, dtype, None), groups, act)


@pytest.mark.parametrize("n,s,c,groups", [(5000, 10, 24, 3), (3000, 3, 8, 2), (1500, 40, 32, 4), (700, 64, 64, 8), (300, 300, 48, 4)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
def test_many_samples(ops, n, s, c, groups, dtype):
    """Workgroups take many samples in turn, the last ones not all."""
    _check(ops, _inputs(n, s, c, dtype, F32), groups, GELU)


@pytest.mark.parametrize("n,s,c,groups", [(4, 50, 32, 4), (2, 9000, 32, 4)])
def test_large_level(ops, n, s, c, groups):
    """Groups whose mean is thousands of times their deviation."""
    _check(ops, _inputs(n, s, c, level=3000.0), groups, NONE)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("n,s,c,groups", [(1, 60001, 100, 5), (2, 52000, 96, 1), (1, 9000, 960, 10)])
def test_many_pieces(ops, n, s, c, groups, dtype):
    """Samples of more pieces than their groups' workgroups should read."""
    _check(ops, _inputs(n, s, c, dtype, level=10.0), groups, SILU)


@pytest.mark.parametrize("n,s,c,groups", [(6, 40, 32, 4), (2, 9001, 40, 5), (2, 9001, 41, 1)])
def test_constant_and_bad_groups(ops, n, s, c, groups):
    """A constant group has y = act(bias) and a finite gradient; NaN and infinities
    stay in their own sample's group."""
    x = _inputs(n, s, c)
    p = c // groups
    x["x"][0, :, :p] = 2.5
    clean, _ = _run(ops, x, groups, SILU)
    b = x["bias"][:p].double()
    assert torch.allclose(clean[0][0, :, :p].cpu().double(), (b * torch.sigmoid(b)).expand(s, p), rtol=1e-6, atol=1e-6)
    assert all(bool(torch.isfinite(t).all()) for t in clean)
    x["x"][1, s // 2, c - 1] = math.nan
    if groups > 1:
        x["x"][1, 0, 0] = math.inf
    dirty, _ = _run(ops, x, groups, SILU)
    for a, b in zip(clean[:2], dirty[:2]):
        bad = torch.isnan(b).cpu().reshape(n, s, groups, p)
        assert bool(bad[1, :, -1].all()) and bool(bad[1, :, 0].all())
        keep = torch.ones(n, groups, dtype=torch.bool)
        keep[1, [0, -1]] = False
        same = (a == b).cpu().reshape(n, s, groups, p).all(1).all(-1)
        assert bool(same[keep].all())


@pytest.mark.parametrize("polls", [1, 2, 5])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("n,s,c,groups", [(2, 4096, 40, 4), (3, 9001, 64, 8), (1, 3001, 250, 10), (2, 2100, 77, 7)])
def test_members_that_do_not_find_the_others(ops, tune, n, s, c, groups, dtype, polls):
    """Workgroups that share a sample look for each other's values no more than so often
    (1: never): what they do not find they compute themselves."""
    tune("GROUP_POLLS", polls)
    _check(ops, _inputs(n, s, c, dtype, F32), groups, SILU)


def test_repeatable(ops):
    for n, s, c, groups in [(900, 30, 48, 6), (2, 9000, 96, 8)]:
        x = _inputs(n, s, c, BF16, F32)
        first, _ = _run(ops, x, groups, GELU)
        for _ in range(3):
            again, _ = _run(ops, x, groups, GELU)
            assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (False, False, False)])
@pytest.mark.parametrize("n,s,c,groups", [(30, 20, 32, 4), (2, 9000, 32, 4)])
def test_wanted_gradients(ops, n, s, c, groups, need):
    x = _inputs(n, s, c)
    every, _ = _run(ops, x, groups, SILU)
    some, _ = _run(ops, x, groups, SILU, need)
    for wanted, a, b in zip(need, every[1:], some[1:]):
        assert torch.equal(a, b) if wanted else b.numel() == 0


@pytest.mark.parametrize("shape", [(0, 4, 8), (3, 0, 8)])
def test_empty(ops, shape):
    x = torch.empty(shape, device=DEV)
    w = torch.ones(8, device=DEV)
    y, stats = ops.group_norm(x, w, w, 2, SILU, EPS)
    assert y.shape == x.shape and stats.shape == (shape[0], 2, 2)
    gx, gw, gb = ops.group_norm_backward(x, x, stats, w, w, 2, SILU, [True] * 3)
    assert gx.shape == x.shape and not bool(gw.any()) and not bool(gb.any()) and gw.shape == gb.shape == (8,)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("shift", [1, 2, 3, 4])
@pytest.mark.parametrize("n,s,c,groups", [(7, 20, 32, 4), (2, 9000, 32, 4)])
def test_addresses(ops, n, s, c, groups, shift, dtype):
    """Tensors at any element of a buffer: the result is that of an aligned copy to its
    rounding, and nothing beside it is written."""
    x = _inputs(n, s, c, dtype, F32)
    size = n * s * c

    def placed(t):
        buf = torch.zeros(size + 16, dtype=dtype, device=DEV)
        buf[shift:shift + size] = t.flatten().to(DEV)
        return buf[shift:shift + size].view(n, s, c)

    w, b = x["weight"].to(DEV), x["bias"].to(DEV)
    y, stats = ops.group_norm(placed(x["x"]), w, b, groups, SILU, EPS)
    grads = ops.group_norm_backward(placed(x["g"]), placed(x["x"]), stats, w, b, groups, SILU, [True] * 3)
    ref, err = _reference(x, groups, SILU)
    for a, r, e, t in zip([y, *grads], ref, err, [dtype, dtype, F32, F32]):
        assert bool(((a.cpu().double() - r).abs() <= e + UNIT[t] * (r.abs() + e) + TINY[t]).all())


def test_gradient_against_differences():
    """The module's gradients against central differences of its own 64-bit CPU path."""
    from piecewiselinearembeddings_optimized_amd import CudaGroupNorm

    torch.manual_seed(0)
    m = CudaGroupNorm(3, 12, activation="gelu").double()
    with torch.no_grad():
        m.weight.add_(0.2 * torch.randn(12))
        m.bias.add_(0.2 * torch.randn(12))
    x = torch.randn(2, 5, 12, dtype=torch.float64)
    g = torch.randn(2, 5, 12, dtype=torch.float64)
    f = lambda: float((m(x) * g).sum())  # noqa: E731
    dev = CudaGroupNorm(3, 12, activation="gelu").to(DEV)
    dev.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    xd = x.float().to(DEV).requires_grad_()
    (dev(xd) * g.float().to(DEV)).sum().backward()
    with torch.no_grad():
        for t, grad in ((x, xd.grad), (m.weight, dev.weight.grad), (m.bias, dev.bias.grad)):
            flat, h = t.view(-1), 1e-5
            for i in range(0, flat.numel(), 7):
                old = float(flat[i])
                flat[i] = old + h
                up = f()
                flat[i] = old - h
                down = f()
                flat[i] = old
                assert abs(float(grad.view(-1)[i]) - (up - down) / (2 * h)) < 2e-4


def test_module_channels_last_view():
    from piecewiselinearembeddings_optimized_amd import CudaGroupNorm

    m = CudaGroupNorm(4, 32, activation="silu").to(DEV)
    x = torch.randn(3, 32, 9, 7, device=DEV).to(memory_format=torch.channels_last).requires_grad_()
    rows = x.movedim(1, -1)
    assert rows.is_contiguous()
    y = m(rows).movedim(-1, 1)
    ref = torch.nn.functional.silu(torch.nn.functional.group_norm(x.double(), 4, eps=1e-5))
    assert torch.allclose(y.double(), ref, rtol=1e-5, atol=1e-5)
    y.sum().backward()
    assert x.grad.shape == x.shape


def test_refusals(ops):
    x, w = torch.randn(2, 3, 8, device=DEV), torch.ones(8, device=DEV)
    bad = [
        (lambda: ops.group_norm(x.double(), w, w, 2, 0, EPS), "float32, float16, or bfloat16"),
        (lambda: ops.group_norm(x, w.double(), w, 2, 0, EPS), "float32, float16, or bfloat16"),
        (lambda: ops.group_norm(x, w.half(), w, 2, 0, EPS), "one dtype"),
        (lambda: ops.group_norm(x, w[:4], w, 2, 0, EPS), "shape"),
        (lambda: ops.group_norm(x, w, w, 3, 0, EPS), "divide"),
        (lambda: ops.group_norm(x, w, w, 0, 0, EPS), "divide"),
        (lambda: ops.group_norm(x, w, w, 2, 4, EPS), "activation"),
        (lambda: ops.group_norm(x.transpose(0, 1), w, w, 2, 0, EPS), "contiguous"),
        (lambda: ops.group_norm(x[0, 0], w, w, 2, 0, EPS), "shape"),
        (lambda: ops.group_norm(x, w.cpu(), w, 2, 0, EPS), "device"),
    ]
    _, stats = ops.group_norm(x, w, w, 2, 0, EPS)
    bad += [
        (lambda: ops.group_norm_backward(x[:1], x, stats, w, w, 2, 0, [True] * 3), "shape and dtype"),
        (lambda: ops.group_norm_backward(x.half(), x, stats, w, w, 2, 0, [True] * 3), "shape and dtype"),
        (lambda: ops.group_norm_backward(x, x, stats[:1].contiguous(), w, w, 2, 0, [True] * 3), "stats"),
        (lambda: ops.group_norm_backward(x, x, stats, w, w, 4, 0, [True] * 3), "stats"),
    ]
    for call, text in bad:
        with pytest.raises(RuntimeError, match=text):
            call()


@pytest.mark.parametrize("n,s,c,groups", [(2, 9000, 30000, 30), (3, 3001, 20000, 10)])
def test_statistics_of_wide_samples(ops, n, s, c, groups):
    """Many pieces of many channels, where the kernels that join them fill the device; the
    first sample is constant."""
    x = torch.empty(n, s, c, dtype=BF16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(1))
    x[0] = 3.0
    stats = ops.group_norm(x, None, None, groups, NONE, EPS)[1]
    for i in range(n):
        for g in range(groups):
            v = x[i, :, g * (c // groups):(g + 1) * (c // groups)].double()
            m = v.mean()
            rho = ((v - m).square().mean() + EPS).rsqrt()
            size = float(rho * v.abs().mean())
            assert abs(float(stats[i, g, 0] - m)) <= E * float(v.abs().mean()), (i, g)
            assert abs(float(stats[i, g, 1] / rho - 1)) <= E * (1 + size) ** 2, (i, g)


@pytest.mark.parametrize("n,s,c,groups,last", [(33000, 256, 256, 32, 2), (9, 9000, 30000, 30, 1)])
def test_more_than_32_bits_of_elements(ops, n, s, c, groups, last):
    """The last samples behind 2^31 elements, against the same samples alone (whose
    workgroups may take other rows: sums of 2^16 or 2^20 values in another order), and the
    parameters' gradients, which are theirs alone."""
    x = torch.empty(n, s, c, dtype=BF16, device=DEV)
    x[:-last].fill_(1.0)
    x[-last:].normal_(generator=torch.Generator(DEV).manual_seed(1))
    g = torch.zeros_like(x)
    g[-last:].normal_(generator=torch.Generator(DEV).manual_seed(2))
    w, b = torch.linspace(0.5, 1.5, c, device=DEV), torch.linspace(-1, 1, c, device=DEV)
    y, stats = ops.group_norm(x, w, b, groups, SILU, EPS)
    gx, gw, gb = ops.group_norm_backward(g, x, stats, w, b, groups, SILU, [True] * 3)
    xs, gs = x[-last:].clone(), g[-last:].clone()
    del x, g
    ys, ss = ops.group_norm(xs, w, b, groups, SILU, EPS)
    gxs, gws, gbs = ops.group_norm_backward(gs, xs, ss, w, b, groups, SILU, [True] * 3)
    # 32-bit values differ by some 2^-20 of their size, 16-bit ones by one step where that
    # crosses a rounding border; sums of 512 to 9000 terms of about 1
    torch.testing.assert_close(stats[-last:], ss, rtol=2.0 ** -18, atol=2.0 ** -18)
    torch.testing.assert_close(y[-last:], ys, rtol=2.0 ** -7, atol=2.0 ** -16)
    torch.testing.assert_close(gx[-last:], gxs, rtol=2.0 ** -7, atol=2.0 ** -16)
    torch.testing.assert_close(gw, gws, rtol=2.0 ** -14, atol=2.0 ** -10)
    torch.testing.assert_close(gb, gbs, rtol=2.0 ** -14, atol=2.0 ** -10)
    assert torch.isfinite(y[:2]).all() and float(gx[:2].abs().max()) == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("n,s,c,groups", [(2, 300, 520, 1), (1, 800, 1000, 1), (1, 20_000, 1280, 32), (1, 9000, 9000, 3)])
def test_narrow_last_slab(ops, n, s, c, groups, dtype):
    """Rows whose slabs are not of one width: lanes without channels in the last."""
    _check(ops, _inputs(n, s, c, dtype, dtype), groups, SILU)


# held in one workgroup and several a slab, shared, split
FORMS = [(6, 40, 32, 4), (300, 64, 64, 8), (40, 30, 250, 10), (2, 9001, 40, 5), (2, 9001, 41, 1), (8, 4096, 64, 8), (2, 3, 9000, 3),
         (1, 90_001, 1000, 10)]


@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("level", [1.0, 3000.0])
@pytest.mark.parametrize("n,s,c,groups", FORMS)
def test_relu_passes_where_its_output_is_positive(ops, n, s, c, groups, level, dtype):
    """The backward's value before the activation is the forward's, bit for bit: a gradient
    of ones gives the bias as many as outputs are above 0 (whole numbers below 2^24), in
    constant groups too, where that is rounding alone."""
    x = _inputs(n, s, c, dtype, F32, level=level)
    x["x"][0, :, :c // groups] = 2.7
    x["g"] = torch.ones_like(x["g"])
    for bias in (torch.zeros(c), x["bias"]):
        got, _ = _run(ops, x | {"bias": bias}, groups, RELU)
        assert torch.equal(got[3], (got[0] > 0).sum((0, 1)).float())
        assert not bool(got[1][:, :, -(c // groups):][(got[0] > 0).any((1, 2)).logical_not()].any())


@pytest.mark.parametrize("n,s,c,groups", [(6, 40, 32, 4), (300, 64, 64, 8), (40, 30, 250, 10), (2, 9000, 40, 5), (2, 9002, 41, 1),
                                          (8, 4096, 64, 8), (2, 4, 9000, 3), (1, 90_000, 1000, 10)])
def test_sums_are_about_the_mean(ops, n, s, c, groups):
    """Groups whose mean is tens of thousands of deviations: the gradients lose nothing by it.
    x - mean is exact here (the mean a power of 2, deviations in pairs), the statistics are
    given; so a sum of terms is off by 64 roundings of their sizes, as one without a mean."""
    gen = torch.Generator().manual_seed(n + s + c)
    p, level = c // groups, 2.0 ** 15
    d = (torch.randn(n, s // 2, c, generator=gen) * 2 ** 7).round() / 2 ** 7
    d = torch.cat([d, -d], 1)
    x, g = level + d, torch.randn(n, s, c, generator=gen)
    w = 1 + 0.3 * torch.randn(c, generator=gen)
    assert torch.equal(x.double() - level, d.double())
    grouped = lambda t: t.reshape(n, s, groups, p)  # noqa: E731
    rho = (grouped(d.double()).square().mean((1, 3)) + EPS).rsqrt().float()
    stats = torch.stack([torch.full_like(rho, level), rho], -1)
    got = ops.group_norm_backward(g.to(DEV), x.to(DEV), stats.to(DEV), w.to(DEV), torch.zeros(c, device=DEV), groups, NONE,
                                  [True] * 3)
    r = rho.double().repeat_interleave(p, 1)[:, None]
    xh, gw = d.double() * r, g.double() * w.double()
    mean = lambda t: grouped(t).mean((1, 3)).repeat_interleave(p, 1)[:, None]  # noqa: E731
    want = [r * (gw - mean(gw) - xh * mean(gw * xh)), (g * xh).sum((0, 1)), g.double().sum((0, 1))]
    err = [r * (gw.abs() + mean(gw.abs()) + xh.abs() * mean((gw * xh).abs())), (g * xh).abs().sum((0, 1)),
           g.double().abs().sum((0, 1))]
    for name, a, b, e in zip(("dx", "dw", "db"), got, want, err):
        off = (a.cpu().double() - b).abs() / (E * e + TINY[F32])
        assert bool((off <= 1).all()), (name, float(off.max()))


@pytest.mark.parametrize("act", [NONE, RELU, SILU, GELU], ids=["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("n,s,c,groups", [(2, 4096, 40, 4), (3, 9001, 64, 8), (1, 3001, 250, 10), (2, 2100, 77, 7), (1, 5000, 64, 64),
                                          (2, 20_011, 256, 32)])
def test_members_compute_the_same_for_each_other(ops, tune, n, s, c, groups, dtype, act):
    """What a member computes in another's place has the bits that the other publishes, so a
    call's results do not depend on who ran when."""
    from piecewiselinearembeddings_optimized_amd import capi

    assert capi.group_norm_plan(n, s, c, groups, dtype)["form"] == 1
    x = _inputs(n, s, c, dtype, F32, level=3.0)
    want, stats = _run(ops, x, groups, act)
    for polls in (1, 2):
        tune("GROUP_POLLS", polls)
        got, again = _run(ops, x, groups, act)
        for name, a, b in zip(("stats", "y", "dx", "dw", "db"), (again, *got), (stats, *want)):
            assert torch.equal(a, b), (polls, name, float((a.double() - b.double()).abs().max()))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("shift", [0, 1, 2, 3, 8])
@pytest.mark.parametrize("n,s,c,groups", [(7, 20, 32, 4), (5, 3, 7, 7), (2, 9000, 32, 4), (3, 3001, 77, 7), (1, 300, 1000, 10), (2, 3, 9001, 1)])
def test_nothing_beside_the_results_is_written(n, s, c, groups, shift, dtype):
    """Results at any element of a buffer (held, shared and split): what lies before and
    behind each stays, and the values are right."""
    from piecewiselinearembeddings_optimized_amd import capi

    x, mark, edge = _inputs(n, s, c, dtype, dtype), 7.0, 64

    def placed(shape, kind, at=shift, fill=None):
        size = math.prod(shape)
        buf = torch.full((edge + size + edge,), mark, dtype=kind, device=DEV)
        t = buf[edge + at:edge + at + size].view(shape)
        if fill is not None:
            t.copy_(fill)
        return buf, t, at

    inputs = {k: placed(v.shape, dtype, fill=v)[1] for k, v in x.items()}
    y, gx = placed((n, s, c), dtype), placed((n, s, c), dtype)
    gw, gb, stats = placed((c,), dtype), placed((c,), dtype), placed((n, groups, 2), F32, shift // 2 * 2)
    capi.group_norm(inputs["x"], inputs["weight"], inputs["bias"], y[1], stats[1], groups, SILU, EPS)
    capi.group_norm_backward(inputs["g"], inputs["x"], stats[1], inputs["weight"], inputs["bias"], gx[1], gw[1], gb[1], groups, SILU)
    for buf, t, at in (y, gx, gw, gb, stats):
        assert bool((buf[:edge + at] == mark).all()) and bool((buf[edge + at + t.numel():] == mark).all())
    ref, err = _reference(x, groups, SILU)
    for (_, a, _), r, e in zip((y, gx, gw, gb), ref, err):
        assert bool(((a.cpu().double() - r).abs() <= e + UNIT[dtype] * (r.abs() + e) + TINY[dtype]).all())

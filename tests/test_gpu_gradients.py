"""The gradients' norm and clipping on the GPU.  The norm is a 64-bit sum rounded to
32 bits: off by at most half a unit (and a millionth of one).  A clipped value is the
32-bit product with a factor rounded to 32 bits, rounded to its type: 2 * 2^-24 and
half a unit of the type, or half of its least positive value."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
LEAST = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}
INF = math.inf


@pytest.fixture(scope="module")
def package():
    assert torch.cuda.is_available(), "HIP device required"
    import piecewiselinearembeddings_optimized_amd as package

    return package


def _grads(shapes, dtypes, scale=1.0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=gen) * scale).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


def _norm(grads, p):
    wide = [g.double().flatten() for g in grads]
    flat = torch.cat(wide) if wide else torch.zeros(0).double()
    if flat.numel() == 0:
        return 0.0
    if p == INF:
        return float(flat.abs().max())
    return float(flat.abs().sum()) if p == 1.0 else math.sqrt(float((flat * flat).sum()))


def _check_norm(got, grads, p):
    ref = _norm(grads, p)
    assert got.dtype == F32 and got.shape == () and got.device.type == "cuda"
    assert abs(float(got) - ref) <= 2.0 ** -24 * 1.000001 * ref + 2.0 ** -150, (float(got), ref)


def _check_scaled(got, grads, factor):
    for g, a in zip(grads, got):
        ref = g.double() * factor
        off = (a.cpu().double() - ref).abs()
        bound = ref.abs() * (2.0 ** -23 + UNIT[a.dtype] * (1 + 2.0 ** -23)) + LEAST[a.dtype] / 2 + 2.0 ** -149
        assert a.shape == g.shape and bool((off <= bound).all())


SHAPES = [(1,), (3,), (0,), (7, 5), (), (64,), (1000,), (33, 65), (4, 0, 3), (20001,), (5, 17000), (16384,), (128, 128), (2,)]


@pytest.mark.parametrize("p", [2.0, 1.0, INF])
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (F32, BF16, F16)], ids=lambda t: "-".join(str(d)[6:] for d in t))
def test_norm_and_clipping(package, dtypes, p):
    grads = _grads(SHAPES, dtypes)
    dev = [g.to(DEV) for g in grads]
    norm = package.gradient_norm(dev, p)
    _check_norm(norm, grads, p)
    limit = 0.37 * _norm(grads, p)
    factor = limit / (_norm(grads, p) + 1e-6)
    for out in (F32, BF16, F16):
        into = [torch.full_like(g, math.nan, dtype=out) for g in dev]
        assert torch.equal(package.clip_gradients_(dev, limit, p, out=into), norm)
        _check_scaled(into, grads, factor)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, grads))
    assert torch.equal(package.clip_gradients_(dev, limit, p), norm)
    _check_scaled(dev, grads, factor)


@pytest.mark.parametrize("count", [1, 99, 100, 101, 350])
def test_many_tensors(package, count):
    """More tensors than one launch lists."""
    grads = _grads([(1 + 13 * (i % 29),) for i in range(count)], (F32, BF16))
    dev = [g.to(DEV) for g in grads]
    for p in (2.0, INF):
        _check_norm(package.gradient_norm(dev, p), grads, p)
    package.clip_gradients_(dev, 0.5, 2.0)
    _check_scaled(dev, grads, 0.5 / (_norm(grads, 2.0) + 1e-6))


def test_large_tensors(package):
    for dtype in (F32, BF16):
        dev = [torch.randn(n, device=DEV, generator=torch.Generator(DEV).manual_seed(n)).to(dtype)
               for n in (40_000_001, 5, 3_000_000)]
        grads = [g.cpu() for g in dev]
        _check_norm(package.gradient_norm(dev), grads, 2.0)
        package.clip_gradients_(dev, 3.0)
        _check_scaled(dev, grads, 3.0 / (_norm(grads, 2.0) + 1e-6))


@pytest.mark.parametrize("size", [1e30, 1e-30])
def test_range(package, size):
    """Squares beyond and below what 32 bits hold."""
    grads = _grads([(1000,), (5, 77)], (F32,), size)
    dev = [g.to(DEV) for g in grads]
    for p in (2.0, 1.0, INF):
        _check_norm(package.gradient_norm(dev, p), grads, p)
    package.clip_gradients_(dev, 0.25 * _norm(grads, 2.0))
    _check_scaled(dev, grads, 0.25 * _norm(grads, 2.0) / (_norm(grads, 2.0) + 1e-6))


def test_nothing_to_clip(package):
    grads = _grads([(100,), (33, 3)], (F32, BF16))
    dev = [g.to(DEV) for g in grads]
    for limit in (_norm(grads, 2.0) * 1.001, INF):
        package.clip_gradients_(dev, limit)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, grads))
        into = [torch.empty_like(g) for g in dev]
        package.clip_gradients_(dev, limit, out=into)
        assert all(torch.equal(a, b) for a, b in zip(dev, into))
    package.clip_gradients_(dev, 0.0)
    assert not any(bool(g.any()) for g in dev)


@pytest.mark.parametrize("p", [2.0, 1.0, INF])
def test_infinities_and_nan(package, p):
    grads = _grads([(100,), (70,)], (F32, F16))
    for bad, place in ((INF, (0, 3)), (-INF, (1, 69)), (math.nan, (0, 99))):
        dev = [g.to(DEV).clone() for g in grads]
        dev[place[0]][place[1]] = bad
        norm = package.clip_gradients_(dev, 1.0, p)
        if math.isnan(bad):
            assert math.isnan(float(norm)) and all(bool(torch.isnan(g).all()) for g in dev)
        else:
            assert float(norm) == INF
            for i, g in enumerate(dev):
                ref = torch.zeros(g.shape)
                if i == place[0]:
                    ref[place[1]] = math.nan
                assert torch.equal(torch.isnan(g.cpu()), torch.isnan(ref)) and not bool(g.nan_to_num(0.0).any())
    zeros = [torch.zeros(5, device=DEV)]
    assert float(package.clip_gradients_(zeros, 1.0, p)) == 0 and not bool(zeros[0].any())
    both = [torch.full((300,), INF, device=DEV), torch.full((300,), math.nan, device=DEV)]
    assert math.isnan(float(package.gradient_norm(both, p)))


def test_layouts(package):
    """Dense tensors in any order of dimensions, and tensors with gaps between rows."""
    base = _grads([(6, 40), (3, 4, 5), (40, 30), (200,)], (F32,))
    dev = [t.to(DEV) for t in base]
    views = [dev[0].t(), dev[1].permute(2, 0, 1), dev[2][:, :7], dev[3][::3]]
    refs = [v.cpu().clone() for v in views]
    rest = dev[2][:, 7:].cpu().clone(), dev[3].cpu().clone()
    _check_norm(package.gradient_norm(views), refs, 2.0)
    package.clip_gradients_(views, 1.0)
    _check_scaled(views, refs, 1.0 / (_norm(refs, 2.0) + 1e-6))
    assert torch.equal(dev[2][:, 7:].cpu(), rest[0])
    untouched = torch.ones(200, dtype=torch.bool)
    untouched[::3] = False
    assert torch.equal(dev[3].cpu()[untouched], rest[1][untouched])
    wide = torch.ones(5, 1, device=DEV).expand(5, 9)
    assert float(package.gradient_norm([wide], 1.0)) == 45.0
    into = torch.empty(5, 9, device=DEV)
    package.clip_gradients_([wide], 9.0, 1.0, out=[into])
    assert torch.allclose(into, torch.full_like(into, 9 / 45))
    with pytest.raises(RuntimeError):
        package.clip_gradients_([wide], 9.0, 1.0)


@pytest.mark.parametrize("shifts", [(1, 1), (1, 2), (3, 0), (0, 5), (4, 4), (7, 3)])
def test_addresses(package, shifts):
    """Views of one buffer at any element, gradients and outputs at different ones;
    nothing beside them is written."""
    for dtype, out in ((F32, F32), (BF16, BF16), (BF16, F32), (F32, BF16), (F16, F32)):
        n = 40_003
        grads = _grads([(n,)], (dtype,))
        buf = torch.zeros(n + 32, dtype=dtype, device=DEV)
        to = torch.full((n + 32,), 7.0, dtype=out, device=DEV)
        g, o = buf[shifts[0]:shifts[0] + n], to[shifts[1]:shifts[1] + n]
        g.copy_(grads[0].to(DEV))
        package.clip_gradients_([g], 2.0, out=[o])
        _check_scaled([o], grads, 2.0 / (_norm(grads, 2.0) + 1e-6))
        assert bool((to[:shifts[1]] == 7).all()) and bool((to[shifts[1] + n:] == 7).all())
        package.clip_gradients_([g], 2.0)
        _check_scaled([g], grads, 2.0 / (_norm(grads, 2.0) + 1e-6))
        assert not bool(buf[:shifts[0]].any()) and not bool(buf[shifts[0] + n:].any())


def test_given_norm(package):
    """A norm over more than these gradients, as sharded ones have."""
    grads = _grads([(100,), (50, 3)], (F32,))
    dev = [g.to(DEV) for g in grads]
    given = torch.tensor(40.0, device=DEV)
    got = package.clip_gradients_(dev, 2.0, norm=given)
    assert float(got) == 40.0 and got.data_ptr() != given.data_ptr()
    _check_scaled(dev, grads, 2.0 / (40.0 + 1e-6))


def test_parameters(package):
    torch.manual_seed(0)
    layers = torch.nn.Sequential(torch.nn.Linear(30, 50), torch.nn.Linear(50, 20)).to(DEV)
    layers(torch.randn(8, 30, device=DEV)).square().sum().backward()
    grads = [p.grad.cpu().clone() for p in layers.parameters()]
    unused = torch.nn.Parameter(torch.ones(3, device=DEV))
    norm = package.clip_grad_norm_([*layers.parameters(), unused, layers[0].weight], 1.5)
    _check_norm(norm, grads, 2.0)
    _check_scaled([p.grad for p in layers.parameters()], grads, 1.5 / (_norm(grads, 2.0) + 1e-6))
    assert unused.grad is None
    layers[0].bias.grad[0] = math.nan
    kept = layers[1].weight.grad.clone()
    with pytest.raises(RuntimeError, match="not finite"):
        package.clip_grad_norm_(layers.parameters(), 1.0, error_if_nonfinite=True)
    assert torch.equal(kept, layers[1].weight.grad)


def test_repeatable(package):
    dev = [g.to(DEV) for g in _grads([(100_000,), (77, 99), (5,)], (F32, BF16))]
    first = package.gradient_norm(dev, 2.0)
    assert all(torch.equal(first, package.gradient_norm(dev, 2.0)) for _ in range(5))


def test_refusals(package):
    a, b = torch.randn(20, device=DEV), torch.randn(20, device=DEV)
    bad = [
        (lambda: package.clip_gradients_([a, a], 1.0), "share memory"),
        (lambda: package.clip_gradients_([a[:12], a[10:]], 1.0), "share memory"),
        (lambda: package.clip_gradients_([a, b], 1.0, out=[b, torch.empty_like(b)]), "share memory"),
        (lambda: package.clip_gradients_([a[:10], b[:10]], 1.0, out=[a[5:15], torch.empty_like(b[:10])]), "share memory"),
        (lambda: package.clip_gradients_([a], 1.0, out=[]), "every gradient"),
        (lambda: package.clip_gradients_([a], 1.0, out=[b[:10]]), "shape"),
        (lambda: package.clip_gradients_([a.view(4, 5)], 1.0, out=[b.view(5, 4).t()]), "strides"),
        (lambda: package.clip_gradients_([a], -1.0), "negative"),
        (lambda: package.clip_gradients_([a], math.nan), "negative"),
        (lambda: package.clip_gradients_([a], 1.0, 3.0), "norm_type"),
        (lambda: package.gradient_norm([a], -INF), "norm_type"),
        (lambda: package.gradient_norm([a, b.cpu()]), "device"),
        (lambda: package.gradient_norm([a.double()]), "float32, float16, or bfloat16"),
        (lambda: package.gradient_norm([a.to_sparse()]), "Sparse"),
        (lambda: package.clip_gradients_([a], 1.0, norm=torch.ones(1)), "device"),
        (lambda: package.clip_gradients_([a], 1.0, norm=torch.ones(2, device=DEV)), "one float32"),
    ]
    kept = a.clone(), b.clone()
    for call, text in bad:
        with pytest.raises((RuntimeError, NotImplementedError), match=text):
            call()
    assert torch.equal(kept[0], a) and torch.equal(kept[1], b)
    # the same tensor twice has a norm, and an output may be the gradient itself
    assert math.isclose(float(package.gradient_norm([a, a])), math.sqrt(2) * float(a.double().norm()), rel_tol=1e-6)
    package.clip_gradients_([a], 1.0, out=[a])
    assert math.isclose(float(a.double().norm()), 1.0, rel_tol=1e-5)


def test_autograd_sees_the_writes(package):
    """A tensor that a graph has saved is scaled: its backward must not use the new values."""
    for into in (False, True):
        x = torch.randn(20, device=DEV, requires_grad=True)
        s = x.exp()                                  # (its backward reads s)
        target = s.detach()
        package.clip_gradients_([torch.ones_like(target)] if into else [target], 0.1, out=[target] if into else None)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            s.sum().backward()
    with torch.inference_mode():
        g = torch.ones(4, device=DEV)
        package.clip_gradients_([g], 1.0)
    assert torch.allclose(g, torch.full_like(g, 0.5))

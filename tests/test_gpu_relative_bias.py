"""The relative position bias on the GPU.  A forward value is one entry of the table,
rounded once: equal to the last bit.  A gradient is a 32-bit sum in trees: off by at
most 64 * 2^-24 of its terms' absolute sum, and half a unit of a 16-bit type."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
E = 64 * 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "HIP device required"
    import piecewiselinearembeddings_optimized_amd  # noqa: F401  (registers the ops)

    return torch.ops.rtdl_num_embeddings_cuda


def _buckets(rows, far, seed=0):
    """Any row for any distance: no order, no symmetry."""
    gen = torch.Generator().manual_seed(seed + rows + far)
    return torch.randint(0, rows, (2 * far + 1,), generator=gen, dtype=torch.int32)


def _rows(buckets, starts, q, k, offset):
    far = buckets.shape[0] // 2
    first = torch.tensor([offset]) if starts is None else starts.clamp(-2 ** 60, 2 ** 60)
    d = torch.arange(k) - (first[:, None, None] + torch.arange(q)[:, None])
    return buckets[d.clamp(-far, far) + far].long(), d


def _check(ops, heads, q, k, rows=9, far=5, starts=None, offset=None, causal=False, weight=F32, out=F32, buckets=None, seed=0,
           fill=None):
    gen = torch.Generator().manual_seed(seed + heads + 3 * q + 5 * k)
    w = torch.randn(rows, heads, generator=gen).to(weight)
    buckets = _buckets(rows, far, seed) if buckets is None else buckets
    offset = k - q if offset is None else offset
    dev_starts = None if starts is None else starts.to(DEV)
    got = ops.relative_bias(w.to(DEV), buckets.to(DEV), dev_starts, q, k, offset, causal, out)
    r, d = _rows(buckets, starts, q, k, offset)
    none, beyond = r < 0, r >= rows
    ref = w.float()[torch.where(none | beyond, 0, r)]
    ref = torch.where(none[..., None], 0.0, ref)
    ref = torch.where(beyond[..., None], math.nan, ref).movedim(-1, 1)
    if causal:
        ref = torch.where((d > 0)[:, None], -math.inf, ref)
    ref = ref.to(out)
    if starts is None:
        ref = ref[0]
    assert got.shape == ref.shape and got.dtype == out
    torch.testing.assert_close(got.cpu(), ref, rtol=0, atol=0, equal_nan=True)

    g = torch.randn(*ref.shape, generator=gen).to(out)
    if fill is not None:
        g = torch.where((d > 0)[:, None] if starts is not None else (d > 0), fill, g)
    grad = ops.relative_bias_backward(g.to(DEV), buckets.to(DEV), dev_starts, rows, offset, causal, weight)
    lead = g if starts is not None else g[None]
    wide = torch.where((d > 0)[:, None] & causal, 0.0, lead.double())
    flat = wide.movedim(1, -1).reshape(-1, heads)
    place = torch.where(none | beyond, rows, r).reshape(-1)
    exact = torch.zeros(rows + 1, heads, dtype=torch.float64).index_add_(0, place, flat)[:rows]
    size = torch.zeros(rows + 1, heads, dtype=torch.float64).index_add_(0, place, flat.abs())[:rows]
    assert grad.shape == (rows, heads) and grad.dtype == weight
    off = (grad.cpu().double() - exact).abs()
    bound = E * size + UNIT[weight] * (exact.abs() + E * size) + (2.0 ** -25 if weight == F16 else 0)
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-30)).max())
    return got, grad


TYPES = [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16), (BF16, F32), (F32, F16)]


def _ids(v):
    return "-".join(str(t)[6:] for t in v)


@pytest.mark.parametrize("types", TYPES, ids=_ids)
@pytest.mark.parametrize("heads,q,k", [(1, 1, 1), (3, 1, 17), (2, 5, 1), (2, 8, 8), (5, 7, 13), (1, 64, 64), (2, 65, 1024),
                                       (1, 130, 1025), (3, 33, 2050), (2, 200, 131), (1, 9, 5003), (7, 1, 1031)])
def test_sizes(ops, heads, q, k, types):
    for causal in (False, True):
        _check(ops, heads, q, k, causal=causal, weight=types[0], out=types[1], fill=math.nan if causal else None)


@pytest.mark.parametrize("far,rows", [(1, 1), (1, 300), (3, 2), (500, 40), (5000, 70), (2000, 4001)])
@pytest.mark.parametrize("causal", [False, True])
def test_tables(ops, far, rows, causal):
    """Distances nearer and further than the lengths, more rows than a workgroup sums."""
    _check(ops, 3, 150, 900, rows=rows, far=far, causal=causal)
    _check(ops, 2, 1, 3000, rows=rows, far=far, causal=causal, out=BF16)


@pytest.mark.parametrize("offset", [0, -7, 5, 400, -400, 10 ** 6, -10 ** 6, 2 ** 40, -2 ** 60, 2 ** 60])
def test_offsets(ops, offset):
    for causal in (False, True):
        _check(ops, 2, 70, 300, offset=offset, causal=causal, far=50)


@pytest.mark.parametrize("types", TYPES[:3], ids=_ids)
@pytest.mark.parametrize("q,k", [(1, 700), (3, 1029), (40, 90)])
def test_starts(ops, q, k, types):
    """A position for each sample, before, in and behind the keys; the same one twice."""
    starts = torch.tensor([0, 5, k - q, k + 100, -30, 5, 2 ** 62, -2 ** 63])
    for causal in (False, True):
        _check(ops, 3, q, k, starts=starts, causal=causal, far=64, rows=12, weight=types[0], out=types[1])
    _check(ops, 2, q, k, starts=starts[:1], far=9)


def test_rows_without_a_bias_and_beyond_the_table(ops):
    buckets = torch.tensor([-1, 0, 3, 1, 2 ** 31 - 1, 2, -2 ** 31], dtype=torch.int32)
    _check(ops, 3, 20, 30, rows=4, buckets=buckets)
    _check(ops, 3, 20, 30, rows=3, buckets=buckets, causal=True, out=BF16)


@pytest.mark.parametrize("shift", [1, 2, 3, 5, 7])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
def test_addresses(ops, shift, dtype):
    """A gradient at any element of a buffer."""
    h, q, k = 3, 70, 1037
    gen = torch.Generator().manual_seed(shift)
    g = torch.randn(h, q, k, generator=gen).to(dtype)
    buf = torch.full((g.numel() + 16,), math.nan, dtype=dtype, device=DEV)
    buf[shift:shift + g.numel()] = g.flatten().to(DEV)
    buckets = _buckets(9, 40).to(DEV)
    a = ops.relative_bias_backward(buf[shift:shift + g.numel()].view(h, q, k), buckets, None, 9, 30, False, F32)
    b = ops.relative_bias_backward(g.to(DEV), buckets, None, 9, 30, False, F32)
    size = torch.zeros(9, h, dtype=torch.float64)
    r, _ = _rows(buckets.cpu(), None, q, k, 30)
    size.index_add_(0, r.reshape(-1), g.double().abs().movedim(0, -1).reshape(-1, h))
    assert bool(((a - b).abs().cpu().double() <= 2 * E * size).all())


@pytest.mark.parametrize("bidirectional", [False, True])
@pytest.mark.parametrize("buckets,far", [(32, 128), (64, 1024), (7, 30), (2, 1), (40, 200), (6, 100_000)])
def test_module(ops, buckets, far, bidirectional):
    from piecewiselinearembeddings_optimized_amd import CudaRelativeBias

    if bidirectional and buckets < 2:
        pytest.skip("a bucket for each side")
    torch.manual_seed(0)
    m = CudaRelativeBias(buckets, 3, max_distance=far, bidirectional=bidirectional, causal=not bidirectional)
    dev = CudaRelativeBias(buckets, 3, max_distance=far, bidirectional=bidirectional, causal=not bidirectional).to(DEV)
    dev.load_state_dict(m.state_dict())
    g = torch.randn(3, 100, 333)
    a, b = m(100, 333), dev(100, 333)
    assert torch.equal(a, b.cpu())
    live = torch.isfinite(a)
    (torch.where(live, a, 0) * g).sum().backward()
    (torch.where(live.to(DEV), b, 0) * g.to(DEV)).sum().backward()
    torch.testing.assert_close(dev.weight.grad.cpu(), m.weight.grad, rtol=1e-4, atol=1e-3)


def test_empty(ops):
    w, buckets = torch.randn(4, 2, device=DEV), _buckets(4, 3).to(DEV)
    for q, k, starts in [(0, 5, None), (5, 0, None), (2, 3, torch.empty(0, dtype=torch.int64, device=DEV))]:
        out = ops.relative_bias(w, buckets, starts, q, k, 0, False, BF16)
        assert out.shape == ((2, q, k) if starts is None else (0, 2, q, k))
        grad = ops.relative_bias_backward(out, buckets, starts, 4, 0, False, F32)
        assert grad.shape == (4, 2) and not bool(grad.any())


def test_repeatable(ops):
    g = torch.randn(4, 300, 3001, device=DEV).bfloat16()
    buckets = _buckets(33, 700).to(DEV)
    first = ops.relative_bias_backward(g, buckets, None, 33, 2000, True, F32)
    for _ in range(3):
        assert torch.equal(first, ops.relative_bias_backward(g, buckets, None, 33, 2000, True, F32))


def test_more_than_32_bits_of_elements(ops):
    """Outputs past 2^32 elements: values and gradient at the far end."""
    h, q, k = 5, 30_001, 30_011        # 4.5e9 elements, 9 GB
    w = torch.randn(7, h, device=DEV)
    buckets = _buckets(7, 20).to(DEV)
    out = ops.relative_bias(w, buckets, None, q, k, 10, False, BF16)
    r, _ = _rows(buckets.cpu(), None, 3, k, 10 + q - 3)
    ref = w.cpu()[r[0]].movedim(-1, 0).bfloat16()
    assert torch.equal(out[:, -3:].cpu(), ref)
    out.zero_()
    out[:, -2:] = 1.0
    grad = ops.relative_bias_backward(out, buckets, None, 7, 10, False, F32)
    count = torch.zeros(7).index_add_(0, r[0, -2:].reshape(-1), torch.ones(2 * k))
    assert torch.equal(grad.cpu(), count[:, None].expand(7, h))
    del out
    torch.cuda.empty_cache()


def test_refusals(ops):
    w, buckets = torch.randn(4, 2, device=DEV), _buckets(4, 3).to(DEV)
    starts = torch.zeros(2, dtype=torch.int64, device=DEV)
    g = torch.randn(2, 3, 5, device=DEV)
    bad = [
        (lambda: ops.relative_bias(w.double(), buckets, None, 3, 5, 0, False, F32), "float32, float16, or bfloat16"),
        (lambda: ops.relative_bias(w, buckets, None, 3, 5, 0, False, torch.float64), "output_dtype"),
        (lambda: ops.relative_bias(w, buckets.long(), None, 3, 5, 0, False, F32), "int32"),
        (lambda: ops.relative_bias(w, buckets[:6], None, 3, 5, 0, False, F32), "far"),
        (lambda: ops.relative_bias(w, buckets[:1], None, 3, 5, 0, False, F32), "far"),
        (lambda: ops.relative_bias(w, buckets.cpu(), None, 3, 5, 0, False, F32), "device"),
        (lambda: ops.relative_bias(w, buckets, starts.int(), 3, 5, 0, False, F32), "int64"),
        (lambda: ops.relative_bias(w, buckets, None, -3, 5, 0, False, F32), "negative"),
        (lambda: ops.relative_bias(w.t(), buckets, None, 3, 5, 0, False, F32), "contiguous"),
        (lambda: ops.relative_bias(w, buckets, None, 3, 5, 2 ** 61, False, F32), "supported range"),
        (lambda: ops.relative_bias_backward(g, buckets, starts, 4, 0, False, F32), "shape"),
        (lambda: ops.relative_bias_backward(g[None], buckets, starts, 4, 0, False, F32), "shape"),
        (lambda: ops.relative_bias_backward(g, buckets, None, 0, 0, False, F32), "num_rows"),
        (lambda: ops.relative_bias_backward(g.double(), buckets, None, 4, 0, False, F32), "float32, float16, or bfloat16"),
    ]
    for call, text in bad:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_gradient_of_more_than_32_bits_of_heads(ops):
    """Samples and heads whose product passes 32 bits, behind which the tensor's last
    elements lie that no whole vector holds."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB")
    n, k = 46_341, 9                                             # n * n * k = 8 * vectors + 1
    g = torch.zeros(n, n, 1, k, dtype=torch.bfloat16, device=DEV)
    g[-1, -1, 0] = torch.arange(1, k + 1)
    g[0, 0, 0] = 1
    buckets = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    starts = torch.full((n,), 4, device=DEV)
    got = ops.relative_bias_backward(g, buckets, starts, 3, 0, False, torch.float32)
    del g
    torch.cuda.empty_cache()
    want = torch.zeros(3, n)
    want[:, 0] = torch.tensor([4.0, 1.0, 4.0])
    want[:, -1] = torch.tensor([1.0 + 2 + 3 + 4, 5, 6 + 7 + 8 + 9])
    assert torch.equal(got.cpu(), want)

"""Embedding lookup and its gradient on the GPU against a 64-bit computation.

Tolerances.  Forward: one product in 32 bits, rounded once to the output's type,
so it is compared bit by bit with the 32-bit product rounded the same way.
Backward: a 32-bit sum of c terms in any order is off its value by at most
c * 2^-24 * sum |g| (first order), scaling and rounding add 2^-24 and half a unit
of the stored type; the bound below has a factor of 2 over that.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "HIP device required"
    import piecewiselinearembeddings_optimized_amd  # noqa: F401  (registers the ops)

    return torch.ops.rtdl_num_embeddings_cuda


def _rows(tokens, v, offsets=None):
    """Table row of every token (-1 missing, -2 beyond), in token order."""
    flat = tokens.reshape(-1).long()
    lo, n = torch.zeros_like(flat), torch.full_like(flat, v)
    if offsets is not None:
        f = torch.arange(flat.numel()) % tokens.shape[-1]
        lo, n = offsets[f], offsets[f + 1] - offsets[f]
    return torch.where(flat < 0, -1, torch.where(flat < n, lo + flat, -2))


def _check_forward(ops, tokens, weight, scale, out_dtype, offsets=None):
    out = ops.lookup(tokens.to(DEV), weight.to(DEV), None if offsets is None else offsets.to(DEV), scale, -1, out_dtype).cpu()
    rows = _rows(tokens, weight.shape[0], offsets)
    expect = (weight.float()[rows.clamp_min(0)] * torch.tensor(scale, dtype=F32)).to(out_dtype)
    expect[rows == -1] = 0
    expect[rows == -2] = float("nan")
    assert out.shape == (*tokens.shape, weight.shape[1]) and out.dtype == out_dtype
    assert torch.equal(torch.nan_to_num(out.reshape(expect.shape), nan=7e4 if out_dtype != F16 else 6e4),
                       torch.nan_to_num(expect, nan=7e4 if out_dtype != F16 else 6e4))


def _check_backward(ops, tokens, grad, v, scale, dtype, offsets=None, padding=-1):
    args = (grad.to(DEV), tokens.to(DEV), None if offsets is None else offsets.to(DEV), v, scale, padding, dtype)
    got = ops.lookup_backward(*args).cpu()
    assert got.shape == (v, grad.shape[-1]) and got.dtype == dtype
    rows = _rows(tokens, v, offsets)
    keep = rows >= 0
    if padding >= 0:
        keep &= tokens.reshape(-1) != padding
    g = grad.reshape(-1, grad.shape[-1]).double()[keep]
    ref = torch.zeros(v, g.shape[1], dtype=torch.float64).index_add_(0, rows[keep], g) * scale
    size = torch.zeros_like(ref).index_add_(0, rows[keep], g.abs()) * abs(scale)
    count = torch.bincount(rows[keep], minlength=v)[:, None].double()
    tiny = 2.0 ** -24 if dtype == F16 else 2.0 ** -126
    bound = 2 * ((count + 2) * 2.0 ** -24 * size + UNIT[dtype] * ref.abs()) + tiny
    off = (got.double() - ref).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    assert bool((got[count[:, 0] == 0] == 0).all())
    again = ops.lookup_backward(*args).cpu()
    assert torch.equal(got.view(torch.uint8), again.view(torch.uint8))      # the same bits every time


PAIRS = [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (BF16, F32)]


@pytest.mark.parametrize("wide", [False, True], ids=["i32", "i64"])
@pytest.mark.parametrize("w,o", PAIRS, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("t,v,d", [(1, 1, 1), (1, 50, 4096), (7, 3, 8), (16, 1000, 512), (33, 17, 15), (130, 300, 100),
                                   (5, 9, 250), (64, 11, 5120)])
def test_forward(ops, t, v, d, w, o, wide):
    gen = torch.Generator().manual_seed(t * d)
    tokens = torch.randint(-1, v + 1, (t,), generator=gen)
    tokens[0] = v - 1
    weight = torch.randn(v, d, generator=gen).to(w)
    _check_forward(ops, tokens if wide else tokens.int(), weight, 3.7, o)


CASES = {
    "one": (1, 1, 1), "one_wide": (1, 40, 4096), "few": (3, 5, 8), "odd": (77, 13, 15), "pairs": (300, 1000, 250),
    "chunk": (32, 4, 64), "chunk_and_one": (33, 4, 64), "tile": (1024, 100, 32), "tile_and_one": (1025, 1023, 16),
    "one_pass": (5000, 1022, 24), "two_passes": (5000, 1024, 24), "vocabulary": (4099, 50257, 72),
    "large_vocabulary": (2000, 300_007, 8), "three_passes": (3000, 2_000_003, 4), "wide": (513, 999, 1032),
    "many": (70_001, 500, 12), "very_wide": (40, 30, 8200),
}


@pytest.mark.parametrize("spread", ["even", "few_rows", "one_row"])
@pytest.mark.parametrize("name", list(CASES))
def test_backward(ops, name, spread):
    t, v, d = CASES[name]
    gen = torch.Generator().manual_seed(t + v)
    high = {"even": v, "few_rows": min(v, 3), "one_row": 1}[spread]
    tokens = torch.randint(0, high, (t,), generator=gen) + (v - high)       # the last rows
    tokens = torch.where(torch.rand(t, generator=gen) < 0.05, -1, tokens)
    g = torch.randn(t, d, generator=gen)
    _check_backward(ops, tokens, g, v, 1.0, F32)
    if v < 100_000:
        _check_backward(ops, tokens.int(), g.bfloat16(), v, d ** 0.5, BF16)


# tokens, rows, width; the sort's passes and bits a pass; whether one workgroup sorts
SORTS = [
    (5120, 1000, 24, 1, 10, True), (5121, 1000, 24, 1, 10, True), (8192, 1000, 24, 1, 10, True), (8193, 1000, 24, 1, 10, False),
    (8191, 70_001, 16, 2, 9, True), (8192, 700_000, 8, 2, 10, True), (8193, 700_000, 8, 2, 10, False),
    (8192, 200, 40, 1, 8, True), (8193, 200, 40, 1, 8, False), (8192, 1_100_003, 4, 3, 7, True),
    (20_000, 70_001, 24, 2, 9, False), (20_000, 131_072, 9, 2, 9, False), (20_000, 60_000, 33, 2, 8, False),
    (20_000, 1_100_003, 4, 3, 7, False), (70_001, 20_000_003, 2, 3, 9, False), (600_000, 900_001, 3, 2, 10, False),
]


@pytest.mark.parametrize("spread", ["even", "few_rows", "one_row"])
@pytest.mark.parametrize("t,v,d,passes,bits,one", SORTS)
def test_sorts(ops, t, v, d, passes, bits, one, spread):
    """Both sorts at their borders, by every number of passes and both shapes of their workgroups."""
    from piecewiselinearembeddings_optimized_amd import capi

    plan = capi.lookup_backward_plan(t, v, d)
    assert (plan["passes"], plan["digit_bits"], bool(plan["one_workgroup"])) == (passes, bits, one)
    gen = torch.Generator().manual_seed(t + v)
    high = {"even": v, "few_rows": min(v, 3), "one_row": 1}[spread]
    tokens = torch.randint(0, high, (t,), generator=gen) + (v - high)
    tokens = torch.where(torch.rand(t, generator=gen) < 0.05, -1, tokens)
    _check_backward(ops, tokens, torch.randn(t, d, generator=gen), v, 1.0, F32)


@pytest.mark.parametrize("w,o", PAIRS, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("d", [1, 6, 15, 64, 520])
def test_backward_types(ops, d, w, o):
    gen = torch.Generator().manual_seed(d)
    tokens = (torch.rand(3001, generator=gen) ** 3 * 211).long()
    tokens[17], tokens[18] = 211, 1 << 40           # beyond the table
    _check_backward(ops, tokens, torch.randn(3001, d, generator=gen).to(o), 211, 0.3, w)


def test_long_runs(ops):
    """Runs over hundreds of chunks, alone and between short ones."""
    tokens = torch.cat([torch.full((20_000,), 7), torch.arange(40) % 5, torch.full((33_333,), 2), torch.full((1,), 9)])
    tokens = tokens[torch.randperm(len(tokens), generator=torch.Generator().manual_seed(1))]
    _check_backward(ops, tokens, torch.randn(len(tokens), 20, generator=torch.Generator().manual_seed(2)), 12, 1.0, F32)


def test_only_missing_tokens_and_none(ops):
    _check_backward(ops, torch.full((500,), -1), torch.randn(500, 16), 30, 2.0, F32)
    _check_backward(ops, torch.zeros(0, dtype=torch.int64), torch.zeros(0, 16), 30, 2.0, BF16)
    assert ops.lookup(torch.zeros(0, 3, dtype=torch.int64, device=DEV), torch.ones(4, 6, device=DEV), None, 1.0, -1,
                      F32).shape == (0, 3, 6)


@pytest.mark.parametrize("d,w", [(32, F32), (15, F32), (16, BF16)])
def test_columns(ops, d, w):
    """Categorical columns: one table a column, missing and unknown categories."""
    gen = torch.Generator().manual_seed(d)
    cards = torch.tensor([2, 1, 300, 17, 5])
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), cards.cumsum(0)])
    tokens = (torch.rand(777, 5, generator=gen) * (cards + 1)).long() - (torch.rand(777, 5, generator=gen) < 0.1).long()
    v = int(cards.sum())
    _check_forward(ops, tokens, torch.randn(v, d, generator=gen).to(w), 1.5, w, offsets)
    g = torch.randn(777, 5, d, generator=gen).to(w)
    _check_backward(ops, tokens, g, v, 1.5, w, offsets)
    _check_backward(ops, tokens.int(), g, v, 1.5, w, offsets, padding=1)


@pytest.mark.parametrize("n,cards", [(1638, [2, 1, 300, 17, 5]), (1639, [2, 1, 300, 17, 5]), (9001, [3, 7000, 40]),
                                     (5000, [70_000, 2, 1, 900]), (3000, [5] * 40), (2000, [400_000, 11, 700_000, 3, 9])])
@pytest.mark.parametrize("d,w", [(32, F32), (10, BF16)])
def test_many_rows_of_columns(ops, n, cards, d, w):
    """Categorical columns beyond what one workgroup sorts."""
    gen = torch.Generator().manual_seed(n + d)
    cards = torch.tensor(cards)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), cards.cumsum(0)])
    u = torch.rand(n, len(cards), generator=gen) ** 2
    tokens = (u * (cards + 0.02)).long() - (torch.rand(n, len(cards), generator=gen) < 0.05).long()
    tokens[7, -1] = int(cards[-1])                  # beyond its column, not beyond the table's others
    tokens[8, 0] = int(cards[0])
    v = int(cards.sum())
    _check_forward(ops, tokens, torch.randn(v, d, generator=gen).to(w), 1.5, w, offsets)
    g = torch.randn(n, len(cards), d, generator=gen).to(w)
    _check_backward(ops, tokens, g, v, 1.5, w, offsets)
    _check_backward(ops, tokens.int(), g, v, 1.5, w, offsets, padding=1)


def test_padding_has_no_gradient(ops):
    gen = torch.Generator().manual_seed(3)
    tokens = torch.randint(0, 6, (400,), generator=gen)
    _check_backward(ops, tokens, torch.randn(400, 24, generator=gen), 6, 1.0, F32, padding=0)


def test_non_finite_gradients_stay_in_their_row(ops):
    tokens = torch.arange(200) % 10
    g = torch.ones(200, 8)
    g[13] = float("inf")
    g[27, 4] = float("nan")
    got = ops.lookup_backward(g.to(DEV), tokens.to(DEV), None, 10, 1.0, -1, F32).cpu()
    assert torch.isinf(got[3]).all() and torch.isnan(got[7, 4]) and got.isfinite().sum() == 80 - 8 - 1


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_unaligned_tensors(ops, dtype):
    """Rows of whole vectors at addresses that are not aligned for them."""
    gen = torch.Generator().manual_seed(4)
    base = torch.randn(50 * 64 + 1, generator=gen).to(dtype)
    tokens = torch.randint(0, 50, (90,), generator=gen)
    weight = base.to(DEV)[1:].view(50, 64)
    out = ops.lookup(tokens.to(DEV), weight, None, 1.0, -1, dtype).cpu()
    assert torch.equal(out, base[1:].view(50, 64)[tokens])
    gbase = torch.randn(90 * 64 + 1, generator=gen).to(dtype)
    got = ops.lookup_backward(gbase.to(DEV)[1:].view(90, 64), tokens.to(DEV), None, 50, 1.0, -1, dtype)
    same = ops.lookup_backward(gbase[1:].clone().to(DEV).view(90, 64), tokens.to(DEV), None, 50, 1.0, -1, dtype)
    assert torch.equal(got, same)


def test_offsets_beyond_32_bits(ops):
    """A table of more than 2^32 elements: its last rows are read and written."""
    v, d = 1_100_000, 4096
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    weight = torch.zeros(v, d, dtype=BF16, device=DEV)
    weight[-1] = 3.0
    weight[v // 2 + 5] = 2.0
    tokens = torch.tensor([v - 1, 0, v // 2 + 5, v - 1], device=DEV)
    out = ops.lookup(tokens, weight, None, 0.5, -1, BF16)
    assert torch.equal(out[:, 0].float().cpu(), torch.tensor([1.5, 0.0, 1.0, 1.5]))
    del weight, out
    g = torch.ones(4, d, dtype=BF16, device=DEV)
    dw = ops.lookup_backward(g, tokens, None, v, 1.0, -1, BF16)
    assert torch.equal(dw[tokens, -1].float().cpu(), torch.tensor([2.0, 1.0, 1.0, 2.0]))
    dw[tokens] = 0
    assert not bool(dw.any())


@pytest.mark.parametrize("t", [4000, 20_000])
def test_clearing_wide_rows_of_a_large_table(ops, t):
    """More rows of over 16 KB than a launch has workgroups to clear them: several rows a workgroup."""
    v, d = 2_100_001, 8200
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    gen = torch.Generator().manual_seed(t)
    rows = torch.randint(0, v, (600,), generator=gen)
    rows[:2] = torch.tensor([0, v - 1])
    tokens = rows[torch.randint(0, 600, (t,), generator=gen)].to(DEV)
    g = torch.randint(-3, 4, (t, d), generator=gen).to(BF16).to(DEV)
    dw = ops.lookup_backward(g, tokens, None, v, 1.0, -1, BF16)
    seen, where = tokens.unique(return_inverse=True)
    want = torch.zeros(len(seen), d, device=DEV).index_add_(0, where, g.float())        # (whole numbers: exact)
    assert torch.equal(dw[seen], want.to(BF16))
    dw[seen] = 0
    assert not any(bool(dw[a:a + 300_000].any()) for a in range(0, v, 300_000))


def test_other_stream(ops):
    tokens = torch.randint(0, 100, (5000,), device=DEV)
    weight = torch.randn(100, 64, device=DEV)
    g = torch.randn(5000, 64, device=DEV)
    want = ops.lookup(tokens, weight, None, 2.0, -1, F32), ops.lookup_backward(g, tokens, None, 100, 2.0, -1, F32)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.lookup(tokens, weight, None, 2.0, -1, F32), ops.lookup_backward(g, tokens, None, 100, 2.0, -1, F32)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graph_replay(ops):
    """A captured forward and backward, replayed with other tokens."""
    tokens = torch.randint(0, 100, (3000,), device=DEV)
    weight, g = torch.randn(100, 32, device=DEV), torch.randn(3000, 32, device=DEV)

    def both():
        return ops.lookup(tokens, weight, None, 2.0, -1, F32), ops.lookup_backward(g, tokens, None, 100, 2.0, -1, F32)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for k in range(4):
        tokens.copy_(torch.randint(0, 100 - 20 * k, (3000,)))
        graph.replay()
        torch.cuda.synchronize()
        want = both()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k


def test_module_gradient_and_differences(ops):
    """Module autograd: the gradient against the formula's on the CPU, and against differences."""
    from piecewiselinearembeddings_optimized_amd import CudaCategoricalEmbeddings, CudaTokenEmbeddings

    torch.manual_seed(0)
    for module, tokens in ((CudaTokenEmbeddings(40, 12, scale=3.0, padding_idx=2), torch.randint(-1, 40, (6, 9))),
                           (CudaCategoricalEmbeddings([3, 30, 7], 10), torch.stack(
                               [torch.randint(-1, c, (50,)) for c in (3, 30, 7)], -1))):
        up = torch.randn(*tokens.shape, module.weight.shape[1])
        want = torch.autograd.grad((module(tokens) * up).sum(), module.weight)[0]
        module = module.to(DEV)
        out = module(tokens.to(DEV))
        got = torch.autograd.grad((out * up.to(DEV)).sum(), module.weight)[0]
        torch.testing.assert_close(got.cpu(), want, rtol=1e-5, atol=1e-5)
        # linear in the weights: one difference of any size is the gradient
        step = torch.randn_like(module.weight)
        if getattr(module, "padding_idx", None) is not None:
            step[module.padding_idx] = 0
        with torch.no_grad():
            before = (out.double() * up.to(DEV)).sum()
            module.weight += step
            after = (module(tokens.to(DEV)).double() * up.to(DEV)).sum()
        assert abs(float(after - before) - float((got.double() * step).sum())) < 1e-3


def test_opcheck(ops):
    weight = torch.randn(20, 8, device=DEV, requires_grad=True)
    tokens = torch.randint(0, 20, (5, 3), device=DEV)
    offsets = torch.tensor([0, 5, 11, 20], device=DEV)
    torch.library.opcheck(ops.lookup.default, (tokens, weight, None, 2.0, 1, F32))
    torch.library.opcheck(ops.lookup.default, (tokens % 5, weight, offsets, 2.0, -1, BF16))


def test_compiled(ops):
    from piecewiselinearembeddings_optimized_amd import CudaTokenEmbeddings

    m = CudaTokenEmbeddings(30, 16, scale=4.0).to(DEV)
    tokens = torch.randint(0, 30, (50,), device=DEV)
    run = torch.compile(lambda t: m(t) * 2, fullgraph=True)
    got = torch.autograd.grad(run(tokens).square().sum(), m.weight)[0]
    want = torch.autograd.grad((m(tokens) * 2).square().sum(), m.weight)[0]
    torch.testing.assert_close(got, want)


def test_refusals(ops):
    w, t = torch.randn(5, 4, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    g = torch.zeros(3, 4, device=DEV)
    for match, call in {
        "int32 or int64": lambda: ops.lookup(t.float(), w, None, 1.0, -1, F32),
        "shape \\[V, D\\]": lambda: ops.lookup(t, w[0], None, 1.0, -1, F32),
        "contiguous": lambda: ops.lookup(t, w.T, None, 1.0, -1, F32),
        "weight must be float32, float16, or bfloat16": lambda: ops.lookup(t, w.double(), None, 1.0, -1, F32),
        "output_dtype must be": lambda: ops.lookup(t, w, None, 1.0, -1, torch.float64),
        "same CUDA device": lambda: ops.lookup(t.cpu(), w, None, 1.0, -1, F32),
        "last dimension of tokens": lambda: ops.lookup(t, w, torch.tensor([0, 2, 5], device=DEV), 1.0, -1, F32),
        "offsets must be int64": lambda: ops.lookup(t, w, torch.tensor([0, 1, 2, 5], device=DEV).int(), 1.0, -1, F32),
        "shape of tokens": lambda: ops.lookup_backward(g[:2], t, None, 5, 1.0, -1, F32),
        "num_rows must be positive": lambda: ops.lookup_backward(g, t, None, 0, 1.0, -1, F32),
        "grad_dtype must be": lambda: ops.lookup_backward(g, t, None, 5, 1.0, -1, torch.int32),
    }.items():
        with pytest.raises(RuntimeError, match=match):
            call()


def test_c_abi(ops):
    """The ctypes binding gives the operators' bits, and refuses a small workspace."""
    from piecewiselinearembeddings_optimized_amd import capi

    gen = torch.Generator(DEV).manual_seed(0)
    tokens = torch.randint(0, 70, (900,), device=DEV, generator=gen)
    weight, g = torch.randn(70, 40, device=DEV, generator=gen), torch.randn(900, 40, device=DEV, generator=gen)
    out, dw = torch.empty_like(g), torch.empty_like(weight)
    capi.lookup(tokens, weight, out, scale=0.5)
    capi.lookup_backward(g, tokens, dw, scale=0.5)
    assert torch.equal(out, ops.lookup(tokens, weight, None, 0.5, -1, F32))
    assert torch.equal(dw, ops.lookup_backward(g, tokens, None, 70, 0.5, -1, F32))
    with pytest.raises(capi.PleError, match="workspace"):
        capi.lookup_backward(g, tokens, dw, workspace=torch.empty(64, dtype=torch.uint8, device=DEV))


@pytest.mark.parametrize("t,d,dtype", [(20_000, 512, BF16), (20_000, 500, BF16), (9000, 1001, F32), (300_000, 16, F32),
                                       (600_000, 4, F32), (1_100_000, 2, BF16)])
def test_workspace_and_steps(ops, t, d, dtype):
    """Chunk lengths above the smallest, and sorts of several steps a workgroup; one workspace size for every layout."""
    gen = torch.Generator().manual_seed(t)
    v = 5001
    tokens = (torch.rand(t, generator=gen) ** 4 * v).long()
    g = torch.randn(t, d, generator=gen).to(dtype)
    _check_backward(ops, tokens, g, v, 1.0, dtype)


def test_more_blocks_than_one_grid(ops):
    """70 million tokens of odd rows beyond one wave: their lanes pass 32 bits."""
    n, d = 70_000_000, 65
    weight = torch.arange(3 * d, dtype=F32).reshape(3, d).to(F16).to(DEV)
    tokens = (torch.arange(n, device=DEV, dtype=torch.int32) * 7) % 3
    tokens[-1] = -1
    out = ops.lookup(tokens, weight, None, 1.0, -1, F16)
    assert not bool(out[-1].any())
    at = torch.cat([torch.arange(0, n - 1, 997), torch.arange(33_554_000, 33_555_000), torch.arange(n - 3000, n - 1)]).to(DEV)
    assert torch.equal(out[at], weight[tokens[at].long()])

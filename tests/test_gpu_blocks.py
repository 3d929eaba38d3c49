"""Group norm, relative bias and gradient clipping as they are used: together, on other
streams, two calls at once, in captured graphs, through the C ABI, compiled.

What is compared with the same kernels on the same values is compared bit for bit:
their sums have a fixed order.
"""

from __future__ import annotations

import copy

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SILU, GELU = 2, 3

# a sample's groups in one workgroup, in several, and in pieces
GROUPS = [(9, 40, 32, 4), (2, 9000, 64, 8), (1, 60001, 100, 5)]


@pytest.fixture(scope="module")
def package():
    assert torch.cuda.is_available(), "HIP device required"
    import piecewiselinearembeddings_optimized_amd as p

    return p


@pytest.fixture(scope="module")
def ops(package):
    return torch.ops.rtdl_num_embeddings_cuda


def _rand(*shape, seed=0, dtype=F32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(dtype).to(DEV)


def _group_case(ops, n, s, c, groups, dtype=F32, seed=0):
    x, g = _rand(n, s, c, seed=seed, dtype=dtype), _rand(n, s, c, seed=seed + 1, dtype=dtype)
    w, b = _rand(c, seed=seed + 2), _rand(c, seed=seed + 3)

    def run():
        y, stats = ops.group_norm(x, w, b, groups, SILU, 1e-5)
        return [y, stats, *ops.group_norm_backward(g, x, stats, w, b, groups, SILU, [True] * 3)]

    return x, run


def _bias_case(package, ops, heads, q, k, starts=None, seed=0):
    buckets = package.relative_buckets(16, 64).to(DEV)
    w = _rand(16, heads, seed=seed)
    b = [] if starts is None else [starts.numel()]
    g = _rand(*b, heads, q, k, seed=seed + 1)

    def run():
        return [ops.relative_bias(w, buckets, starts, q, k, k - q, True, BF16),
                ops.relative_bias_backward(g, buckets, starts, 16, k - q, True, F32)]

    return w, run


def _clip_case(package, seed=0):
    grads = [_rand(n, seed=seed) for n in (70001, 5, 1, 4096)]
    out = [torch.empty_like(g) for g in grads]

    def run():
        return [package.clip_gradients_(grads, 1.5, out=out), *(o.clone() for o in out)]

    return grads[0], run


def _cases(package, ops, seed=0):
    starts = torch.tensor([3, 0, 200], device=DEV)
    return ([_group_case(ops, *s, dtype=t, seed=seed) for s in GROUPS for t in (F32, BF16)]
            + [_bias_case(package, ops, 4, 1, 700, seed=seed), _bias_case(package, ops, 3, 130, 301, seed=seed),
               _bias_case(package, ops, 2, 65, 90, starts, seed=seed), _clip_case(package, seed)])


def _same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_other_stream(package, ops):
    cases = _cases(package, ops)
    want = [run() for _, run in cases]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = [run() for _, run in cases]
    s.synchronize()
    assert all(_same(a, b) for a, b in zip(got, want))


def test_two_calls_at_once(package, ops):
    """Calls on two streams that share the device: members of two calls' samples run
    and wait for each other side by side."""
    a, b = _cases(package, ops), _cases(package, ops, seed=50)
    want = [[run() for _, run in c] for c in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for k in range(len(a)):
        for side, (c, s) in enumerate(zip((a, b), streams)):
            with torch.cuda.stream(s):
                got[side].append(c[k][1]())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(_same(x, y) for x, y in zip(g, w))


def test_captured(package, ops):
    """Every operator in one graph, replayed with other values; the eager results come
    from between the replays."""
    cases = _cases(package, ops)
    for _, run in cases:
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [run() for _, run in cases]
    for k in range(4):
        for t, _ in cases:
            t.mul_(0.5 + k)
        graph.replay()
        torch.cuda.synchronize()
        kept = [[t.clone() for t in h] for h in held]
        assert all(_same(a, run()) for a, (_, run) in zip(kept, cases)), k


def test_two_graphs_at_once(package, ops):
    """Two captured calls replayed on two streams do not share their workspaces."""
    cases = [_group_case(ops, 2, 9000, 64, 8, seed=s) for s in (0, 50)]
    want = [run() for _, run in cases]
    torch.cuda.synchronize()
    graphs, held = [], []
    for _, run in cases:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(run())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(_same(a, b) for a, b in zip(held, want))


class Model(nn.Module):
    """Numbers -> embeddings -> group norm -> attention with the relative bias -> logits."""

    def __init__(self, package, bins, d=16, heads=2, causal=False):
        super().__init__()
        self.embed = package.CudaPiecewiseLinearEmbeddings(bins, d, activation=False, version="B")
        self.norm = package.CudaGroupNorm(4, d, activation="gelu")
        self.bias = package.CudaRelativeBias(8, heads, max_distance=16, causal=causal)
        self.qkv = nn.Linear(d, 3 * d)
        self.head = nn.Linear(d, 1)
        self.heads = heads

    def forward(self, x):
        e = self.embed(x)
        n, f, d = e.shape
        q, k, v = self.qkv(self.norm(e)).view(n, f, 3, self.heads, -1).permute(2, 0, 3, 1, 4)
        scores = (q.unsqueeze(-2) * k.unsqueeze(-3)).sum(-1) * (d // self.heads) ** -0.5 + self.bias(f)
        a = (torch.softmax(scores, -1).unsqueeze(-1) * v.unsqueeze(-3)).sum(-2)
        return self.head(e + a.transpose(1, 2).reshape(n, f, d)).mean((1, 2))


def _model(package, causal=False):
    torch.manual_seed(3)
    x = torch.randn(96, 7)
    bins = package.compute_bins(x, n_bins=12)
    return Model(package, bins, causal=causal), x


def _gradients(model, x, limit, package):
    for p in model.parameters():
        p.grad = None
    loss = model(x).square().mean()
    loss.backward()
    norm = package.clip_grad_norm_(model.parameters(), limit)
    return [loss.detach(), norm, *(p.grad for p in model.parameters() if p.grad is not None)]


@pytest.mark.parametrize("causal", [False, True])
def test_together(package, causal):
    """A training step's loss, norm and clipped gradients, against the CPU's plain
    operations.  Both compute in 32 bits; a gradient is a sum over 96 * 7 rows of a
    chain of some twenty operations, each off by a few 2^-24 of sums of at most 16
    terms: 2^-24 * 20 * 16 * 4 = 8e-5 of the largest gradient, the loss and norm alike."""
    model, x = _model(package, causal)
    limit = 0.05
    want = _gradients(model, x, limit, package)
    got = _gradients(copy.deepcopy(model).to(DEV), x.to(DEV), limit, package)
    assert float(want[1]) > limit
    largest = max(float(t.abs().max()) for t in want[2:])
    for a, b in zip(got, want):
        torch.testing.assert_close(a.cpu(), b, rtol=1e-4, atol=1e-4 * largest)


def test_together_captured(package):
    model, x = _model(package)
    model, x = model.to(DEV), x.to(DEV)
    params = list(model.parameters())
    norms = torch.empty(2, device=DEV)

    def step():
        loss = model(x).square().mean()
        grads = [g for g in torch.autograd.grad(loss, params, allow_unused=True) if g is not None]
        norms[0] = package.clip_gradients_(grads, 0.05)
        return [loss.detach(), *grads]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        held = step()
    for k in range(3):
        with torch.no_grad():
            for p in params:
                p.mul_(1.1)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*held, norms[0])]
        want = [*step(), norms[0]]
        for a, b in zip(got, want):
            torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)


def test_compiled(package, ops):
    x, w, b = _rand(6, 9, 16), _rand(16, seed=1), _rand(16, seed=2)
    table, buckets = _rand(8, 2), package.relative_buckets(8, 16).to(DEV)

    def step(x, w, b, table):
        y = ops.group_norm(x, w, b, 4, GELU, 1e-5)[0]
        scores = torch.softmax(ops.relative_bias(table, buckets, None, 9, 9, 0, True, F32), -1)
        return (y[:, None] * scores.sum(0)[0, :, None]).sum() + (scores[..., 0] ** 2).sum()

    leaves = [t.requires_grad_() for t in (x, w, b, table)]
    want = torch.autograd.grad(step(*leaves), leaves)
    got = torch.autograd.grad(torch.compile(step, backend="aot_eager", fullgraph=True)(*leaves), leaves)
    for a, c in zip(got, want):
        torch.testing.assert_close(a, c, rtol=1e-5, atol=1e-5)


def test_opcheck(package, ops):
    x, g = _rand(5, 6, 8), _rand(5, 6, 8, seed=1)
    w, b = _rand(8, seed=2).requires_grad_(), _rand(8, seed=3).requires_grad_()
    torch.library.opcheck(ops.group_norm.default, (x.clone().requires_grad_(), w, b, 2, SILU, 1e-5))
    stats = ops.group_norm(x, None, None, 2, SILU, 1e-5)[1]
    torch.library.opcheck(ops.group_norm_backward.default, (g, x, stats, w.detach(), b.detach(), 2, SILU, [True] * 3))
    buckets = package.relative_buckets(8, 16).to(DEV)
    starts = torch.tensor([4, 0], device=DEV)
    table = _rand(8, 3).requires_grad_()
    torch.library.opcheck(ops.relative_bias.default, (table, buckets, None, 5, 9, 4, True, F16),
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    torch.library.opcheck(ops.relative_bias.default, (table, buckets, starts, 5, 9, 0, False, F32))
    torch.library.opcheck(ops.relative_bias_backward.default, (_rand(2, 3, 5, 9), buckets, starts, 8, 0, True, F32))
    grads = [_rand(30), _rand(7, seed=1)]
    torch.library.opcheck(ops.gradient_norm.default, (grads, 2.0))
    torch.library.opcheck(ops.clip_gradients_.default, (grads, 0.5, 2.0, None))
    torch.library.opcheck(ops.clip_gradients_into.default, (grads, [t.clone() for t in grads], 0.5, 2.0, None))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("n,s,c,groups", GROUPS)
def test_c_abi_group_norm(ops, n, s, c, groups, dtype):
    """The same bits as the operators', in a workspace of just the size that is asked for."""
    from piecewiselinearembeddings_optimized_amd import capi

    x, g = _rand(n, s, c, dtype=dtype), _rand(n, s, c, seed=1, dtype=dtype)
    w, b = _rand(c, seed=2), _rand(c, seed=3)
    y, stats = torch.empty_like(x), torch.empty(n, groups, 2, device=DEV)
    gx, gw, gb = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    capi.group_norm(x, w, b, y, stats, groups, SILU)
    capi.group_norm_backward(g, x, stats, w, b, gx, gw, gb, groups, SILU)
    want = ops.group_norm(x, w, b, groups, SILU, 1e-5)
    want = [*want, *ops.group_norm_backward(g, x, want[1], w, b, groups, SILU, [True] * 3)]
    assert _same([y, stats, gx, gw, gb], want)
    size = capi.lib().ple_group_norm_backward_workspace_bytes(n, s, c, groups, capi.dtype_code(dtype))
    assert size > 0
    with pytest.raises(capi.PleError, match="workspace"):
        capi.group_norm_backward(g, x, stats, w, b, gx, gw, gb, groups, SILU,
                                 workspace=torch.empty(size - 1, dtype=torch.uint8, device=DEV))


@pytest.mark.parametrize("q,k,starts", [(1, 300, None), (70, 200, None), (33, 40, [5, 0])])
def test_c_abi_relative_bias(package, ops, q, k, starts):
    from piecewiselinearembeddings_optimized_amd import capi

    starts = None if starts is None else torch.tensor(starts, device=DEV)
    lead = () if starts is None else (2,)
    buckets, w = package.relative_buckets(8, 16).to(DEV), _rand(8, 3)
    g, out, gw = _rand(*lead, 3, q, k), torch.empty(*lead, 3, q, k, device=DEV, dtype=BF16), torch.empty(8, 3, device=DEV)
    capi.relative_bias(w, buckets, out, starts, 7, True)
    capi.relative_bias_backward(g, buckets, gw, starts, 7, True)
    assert torch.equal(out, ops.relative_bias(w, buckets, starts, q, k, 7, True, BF16))
    assert torch.equal(gw, ops.relative_bias_backward(g, buckets, starts, 8, 7, True, F32))
    size = capi.lib().ple_relative_bias_backward_workspace_bytes(max(1, len(lead) * 2), 3, q, k, 8, buckets.numel() // 2)
    if size > 0:
        with pytest.raises(capi.PleError, match="workspace"):
            capi.relative_bias_backward(g, buckets, gw, starts, 7, True,
                                        workspace=torch.empty(size - 1, dtype=torch.uint8, device=DEV))


@pytest.mark.parametrize("kind,p", [(1, 1.0), (2, 2.0), (3, float("inf"))])
def test_c_abi_gradients(package, kind, p):
    from piecewiselinearembeddings_optimized_amd import capi

    grads = [_rand(9001, dtype=BF16), _rand(3), _rand(40000, seed=1)]
    norm, out = torch.empty((), device=DEV), [torch.empty_like(g, dtype=F32) for g in grads]
    capi.grad_norm(grads, norm, kind)
    capi.grad_scale(grads, norm, 0.5, out)
    want = [torch.empty_like(o) for o in out]
    assert torch.equal(norm, package.clip_gradients_(grads, 0.5, p, out=want))
    assert _same(out, want)
    both, into = torch.empty((), device=DEV), [torch.empty_like(o) for o in out]
    capi.grad_clip(grads, both, 0.5, kind, into)
    assert torch.equal(both, norm) and _same(into, want)
    size = capi.lib().ple_grad_norm_workspace_bytes(*capi.gradient_list(grads))
    with pytest.raises(capi.PleError, match="workspace"):
        capi.grad_norm(grads, norm, kind, workspace=torch.empty(size - 1, dtype=torch.uint8, device=DEV))
    with pytest.raises(capi.PleError, match="workspace"):
        capi.grad_clip(grads, norm, 0.5, kind, into, workspace=torch.empty(size - 1, dtype=torch.uint8, device=DEV))


def test_gradients_with_gaps_that_share_memory(package):
    a = _rand(40)
    kept = a.clone()
    for views in ([a[::2], a[::2]], [a[::2], a[10:20]], [a.view(8, 5)[:, :2], a], [a.view(8, 5)[:, 1:3], a.view(8, 5)[:, 1:2]]):
        with pytest.raises(RuntimeError, match="share memory"):
            package.clip_gradients_(views, 0.5)
    assert torch.equal(a, kept)
    package.clip_gradients_([a[::2], a[1::2]], 0.5)                  # of one tensor, but apart
    torch.testing.assert_close(a, kept * (0.5 / (kept.norm() + 1e-6)))


def test_example_with_clipping():
    from tests.test_example import _example

    run = lambda **kw: _example().train("cuda", steps=3, rows=512, batch=256, report=lambda s: None, **kw)  # noqa: E731
    assert run(clip=float("inf")) == run()
    assert all(map(torch.isfinite, map(torch.tensor, run(clip=0.1))))


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("with_starts", [False, True])
def test_compiled_decoding(package, with_starts, train):
    """A compiled module that gets a key more each time is compiled for the first length, and
    once for all others."""
    bias = package.CudaRelativeBias(8, 2, max_distance=16, bidirectional=False, causal=True).to(DEV)
    starts = torch.tensor([3, 9], device=DEV) if with_starts else None
    graphs = []

    def backend(gm, inputs):
        graphs.append(gm)
        return torch._dynamo.backends.registry.lookup_backend("aot_eager")(gm, inputs)

    torch._dynamo.reset()
    compiled = torch.compile(lambda q, k: bias(q, k, starts=starts) * 2, backend=backend, fullgraph=True)
    for k in range(10, 30):
        with torch.set_grad_enabled(train):
            want, got = bias(1, k, starts=starts) * 2, compiled(1, k)
        assert torch.equal(got, want)
        if train:
            g = _rand(*want.shape)
            assert torch.equal(*(torch.autograd.grad(out, bias.weight, g)[0] for out in (got, want)))
    torch._dynamo.reset()
    assert len(graphs) == 2

"""Group norm, relative position bias and the gradients' clipping without a GPU:
refusals of the C ABI, FakeTensor contracts, autograd formulas (meta tensors), the
buckets, and the CPU path against 64-bit computations."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import piecewiselinearembeddings_optimized_amd as pkg
from piecewiselinearembeddings_optimized_amd import capi

_ops = torch.ops.rtdl_num_embeddings_cuda
F32, BF16, F64 = torch.float32, torch.bfloat16, torch.float64
P, ODD = ctypes.c_void_p(256), ctypes.c_void_p(257)
INF = math.inf


def test_c_abi_refuses_group_norms():
    lib = capi.lib()

    def forward(x=P, w=P, b=P, y=P, st=P, n=2, s=3, c=8, g=2, act=0, t=0, pt=0, ws=None, size=0):
        return lib.ple_group_norm_launch(x, w, b, y, st, n, s, c, g, act, 1e-5, t, pt, ws, size, None)

    def backward(dy=P, x=P, st=P, w=P, b=P, dx=P, dw=P, db=P, n=2, s=3, c=8, g=2, act=0, t=0, pt=0, ws=None, size=0):
        return lib.ple_group_norm_backward_launch(dy, x, st, w, b, dx, dw, db, n, s, c, g, act, t, pt, ws, size, None)

    for call in (forward, backward):
        assert call(n=-1) == call(s=-1) == call(c=0) == call(g=0) == call(g=3) == -2
        assert call(t=5) == call(pt=-1) == -3
        assert call(x=None) == call(st=None) == -1
        assert call(c=1 << 21, g=1) == call(n=1 << 31) == call(s=1 << 31) == call(n=1 << 20, s=1 << 20, c=64) == -5
        assert call(x=ODD) == call(w=ODD) == call(b=ODD) == call(st=ODD) == -8
        assert call(act=4) == call(act=-1)
    assert forward(act=4) == capi.lib().ple_grad_scale_launch(None, 0, P, -1.0, None)       # "unsupported"
    assert forward(n=0) == forward(s=0) == 0 and forward(y=None) == -1 and forward(y=ODD) == -8
    assert backward(dx=None, dw=None, db=None) == 0 and backward(dy=None) == -1
    assert backward(dx=ODD) == backward(dw=ODD) == backward(db=ODD) == -8
    assert backward() == -6                                                                 # no workspace
    assert forward(n=1, s=70_000, c=64) == -6
    assert lib.ple_group_norm_workspace_bytes(2, 3, 8, 3, 0) == lib.ple_group_norm_backward_workspace_bytes(0, 3, 8, 2, 0) == 0
    assert lib.ple_group_norm_workspace_bytes(1, 70_000, 64, 2, 0) > 0


def test_c_abi_refuses_relative_biases():
    lib = capi.lib()

    def forward(w=P, u=P, st=None, o=P, b=1, h=2, q=3, k=4, r=5, far=2, offset=0, t=0, ot=0):
        return lib.ple_relative_bias_launch(w, u, st, o, b, h, q, k, r, far, offset, 0, t, ot, None)

    def backward(g=P, u=P, st=None, w=P, b=1, h=2, q=3, k=4, r=5, far=2, offset=0, t=0, ot=0):
        return lib.ple_relative_bias_backward_launch(g, u, st, w, b, h, q, k, r, far, offset, 0, ot, t, None, 0, None)

    for call in (forward, backward):
        assert call(h=0) == call(q=-1) == call(k=-1) == call(r=0) == call(far=0) == call(b=2) == call(b=-1) == -2
        assert call(t=3) == call(ot=9) == -3
        assert call(u=None) == call(w=None) == -1
        assert call(far=(1 << 24) + 1) == call(q=1 << 31) == call(h=1 << 31) == call(offset=(1 << 60) + 1) == -5
        assert call(b=1 << 20, st=P, h=1 << 10, q=1 << 10, k=1 << 10) == call(r=1 << 30, h=1 << 20) == -5
        assert call(w=ODD) == call(u=ODD) == call(st=ODD) == -8
    assert forward(q=0) == forward(k=0) == forward(b=0) == 0 and forward(o=None) == -1 and forward(o=ODD) == -8
    assert backward(g=None) == -1 and backward(g=ODD) == -8 and backward() == -6
    assert lib.ple_relative_bias_backward_workspace_bytes(1, 2, 3, 4, 5, 0) == 0
    assert lib.ple_relative_bias_backward_workspace_bytes(1, 2, 3, 4, 5, 2) > 0


def test_c_abi_refuses_gradients():
    lib = capi.lib()

    def listed(**kw):
        return (capi.Grad * 1)(capi.Grad(**({"grad": 256, "out": 256, "numel": 4, "dtype": 0, "out_dtype": 0} | kw)))

    def norm(g=None, count=1, kind=2, out=P, ws=P, size=1 << 20):
        return lib.ple_grad_norm_launch(listed() if g is None else g, count, kind, out, ws, size, None)

    def scale(g=None, count=1, n=P, limit=1.0):
        return lib.ple_grad_scale_launch(listed() if g is None else g, count, n, limit, None)

    for call in (norm, scale):
        assert call(count=-1) == call(listed(numel=-1)) == -2
        assert call(listed(numel=(1 << 40) + 1)) == -5
        assert call(listed(dtype=4)) == -3
        assert call(listed(grad=None)) == -1
        assert call(listed(grad=258)) == -8
    assert lib.ple_grad_norm_launch(None, 1, 2, P, P, 1 << 20, None) == -1
    assert norm(out=None) == -1 and norm(out=ODD) == -8 and norm(ws=None) == norm(size=7) == norm(ws=ctypes.c_void_p(264)) == -6
    assert norm(kind=0) == norm(kind=4) == scale(limit=-1.0) == scale(limit=math.nan) == scale(listed(out_dtype=1))
    assert scale(listed(out=None)) == scale(n=None) == -1 and scale(listed(out=514)) == -8 and scale(listed(out_dtype=-1)) == -3
    assert scale(count=0) == 0
    assert lib.ple_grad_norm_workspace_bytes(listed(), 1) >= 8


def test_c_abi_refuses_clipping():
    lib = capi.lib()

    def clip(count=1, kind=2, limit=1.0, out=P, ws=P, size=1 << 20, **kw):
        g = (capi.Grad * 1)(capi.Grad(**({"grad": 256, "out": 256, "numel": 4, "dtype": 0, "out_dtype": 0} | kw)))
        return lib.ple_grad_clip_launch(g, count, kind, limit, out, ws, size, None)

    assert clip(count=-1) == clip(numel=-1) == -2 and clip(numel=(1 << 40) + 1) == -5
    assert clip(dtype=4) == clip(out_dtype=-1) == -3
    assert clip(grad=None) == clip(out=None) == lib.ple_grad_clip_launch(None, 1, 2, 1.0, P, P, 1 << 20, None) == -1
    assert clip(grad=258) == clip(out=ODD) == -8
    assert clip(ws=None) == clip(size=7) == clip(ws=ctypes.c_void_p(264)) == -6
    assert clip(kind=0) == clip(kind=4) == clip(limit=-1.0) == clip(limit=math.nan) == clip(out_dtype=1) == -7


def _meta(*shape, dtype=F32):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_fake_shapes():
    y, stats = _ops.group_norm(_meta(2, 5, 8, dtype=BF16), _meta(8), None, 4, 1, 1e-5)
    assert y.shape == (2, 5, 8) and y.dtype == BF16 and stats.shape == (2, 4, 2) and stats.dtype == F32
    gx, gw, gb = _ops.group_norm_backward(y, y, stats, _meta(8), None, 4, 1, [True, True, True])
    assert gx.shape == y.shape and gw.shape == (8,) and gb.shape == (0,)
    buckets, starts = _meta(9, dtype=torch.int32), _meta(3, dtype=torch.int64)
    assert _ops.relative_bias(_meta(6, 4), buckets, None, 5, 7, 2, True, BF16).shape == (4, 5, 7)
    out = _ops.relative_bias(_meta(6, 4), buckets, starts, 5, 7, 2, True, BF16)
    assert out.shape == (3, 4, 5, 7) and out.dtype == BF16
    assert _ops.relative_bias_backward(out, buckets, starts, 6, 2, True, F32).shape == (6, 4)
    assert _ops.gradient_norm([y, stats], 2.0).shape == () and _ops.clip_gradients_([y], 1.0, 2.0, None).dtype == F32
    with pytest.raises(RuntimeError, match="divide"):
        _ops.group_norm(_meta(2, 5, 8), None, None, 3, 0, 1e-5)
    with pytest.raises(RuntimeError, match="int32"):
        _ops.relative_bias(_meta(6, 4), starts, None, 5, 7, 2, True, BF16)


def _recorded(op):
    if op == "group_norm":
        wrt = [_meta(4, 3, 8).requires_grad_(), _meta(8).requires_grad_(), _meta(8).requires_grad_()]
        return _ops.group_norm(*wrt, 2, 2, 1e-5)[0], wrt
    wrt = [_meta(6, 4).requires_grad_()]
    return _ops.relative_bias(wrt[0], _meta(9, dtype=torch.int32), None, 5, 7, 2, False, F32), wrt


OPS = ["group_norm", "relative_bias"]


@pytest.mark.parametrize("op", OPS)
def test_autograd_formulas(op):
    out, wrt = _recorded(op)
    assert [g.shape for g in torch.autograd.grad(out.sum(), wrt)] == [t.shape for t in wrt]


@pytest.mark.parametrize("op", OPS)
def test_compiled_autograd(op):
    from torch._dynamo import compiled_autograd

    out, wrt = _recorded(op)
    graphs = []
    with compiled_autograd._enable(lambda gm: graphs.append(gm) or gm):
        out.sum().backward()
    assert len(graphs) == 1
    assert [t.grad.shape for t in wrt] == [t.shape for t in wrt]


@pytest.mark.parametrize("op", OPS)
def test_no_forward_mode(op):
    out, wrt = _recorded(op)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(wrt[0].detach(), _meta(*wrt[0].shape)).requires_grad_()
        with pytest.raises(NotImplementedError, match="forward-mode"):
            if op == "group_norm":
                _ops.group_norm(dual, *wrt[1:], 2, 2, 1e-5)
            else:
                _ops.relative_bias(dual, _meta(9, dtype=torch.int32), None, 5, 7, 2, False, F32)


def test_statistics_are_not_differentiable():
    y, stats = _ops.group_norm(_meta(4, 3, 8).requires_grad_(), None, None, 2, 0, 1e-5)
    assert y.requires_grad and not stats.requires_grad


@pytest.mark.parametrize("activation", [None, "relu", "silu", "gelu"])
@pytest.mark.parametrize("shape,groups", [((3, 5, 12), 3), ((2, 12), 4), ((2, 3, 4, 12), 12), ((0, 5, 12), 3), ((2, 0, 12), 3)])
def test_module_group_norm_on_cpu(shape, groups, activation):
    torch.manual_seed(0)
    m = pkg.CudaGroupNorm(groups, 12, activation=activation)
    with torch.no_grad():
        m.weight.add_(torch.randn(12))
        m.bias.add_(torch.randn(12))
    x = torch.randn(shape) + 2
    y = m(x)
    assert y.shape == x.shape
    if x.numel() == 0:
        return
    act = {None: lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[activation]
    ref = act(torch.nn.functional.group_norm(x.double().movedim(-1, 1), groups, m.weight.double(), m.bias.double(), 1e-5))
    torch.testing.assert_close(y.double(), ref.movedim(1, -1), rtol=1e-5, atol=1e-5)
    assert m(x.bfloat16()).dtype == BF16 and m.double()(x.double()).dtype == F64
    assert pkg.CudaGroupNorm(groups, 12, affine=False).weight is None


@pytest.mark.parametrize("buckets,far,bidirectional", [(32, 128, True), (32, 128, False), (40, 200, True), (16, 50, False),
                                                       (64, 1024, False), (7, 30, False), (6, 100_000, True), (1, 1, False)])
def test_buckets(buckets, far, bidirectional):
    """Against the logarithm's formula, away from where its rounding decides."""
    got = pkg.relative_buckets(buckets, far, bidirectional)
    assert got.shape == (2 * far + 1,) and got.dtype == torch.int32
    side = buckets // 2 if bidirectional else buckets
    exact = side // 2
    for d in [*range(min(far, 3000) + 1), far - 1, far]:
        if d < exact or exact == 0:
            want = {d if exact else 0}
        else:
            at = exact + math.log(d / exact) / math.log(far / exact) * (side - exact)
            want = {min(side - 1, math.floor(at + e)) for e in (-1e-9, 1e-9)}
        assert int(got[far - d]) in want, d
        if d > 0:
            assert int(got[far + d]) == (int(got[far - d]) + side if bidirectional else 0)


def test_bucket_borders_are_whole_numbers():
    """8 * 16 ** (j / 8): exactly 16, 32 and 64 at j = 2, 4, 6."""
    got = pkg.relative_buckets(32, 128, True)
    for d, row in ((8, 8), (11, 8), (12, 9), (15, 9), (16, 10), (31, 11), (32, 12), (63, 13), (64, 14), (127, 15), (128, 15)):
        assert int(got[128 - d]) == row and int(got[128 + d]) == 16 + row


def test_module_relative_bias_on_cpu():
    torch.manual_seed(0)
    m = pkg.CudaRelativeBias(8, 3, max_distance=20)
    out = m(4, 9)
    assert out.shape == (3, 4, 9)
    for i in range(4):
        for j in range(9):
            row = int(m.buckets[j - (i + 5) + 20])
            assert torch.equal(out[:, i, j], m.weight[row])
    starts = torch.tensor([5, 0])
    both = m(4, 9, starts=starts)
    assert both.shape == (2, 3, 4, 9) and torch.equal(both[0], out) and torch.equal(both[1], m(4, 9, offset=0))
    causal = pkg.CudaRelativeBias(8, 3, bidirectional=False, causal=True)(5)
    assert torch.equal(torch.isneginf(causal[0]), torch.ones(5, 5).triu(1).bool())
    own = pkg.CudaRelativeBias(2, 1, buckets=torch.tensor([1, -1, 2]))
    out = own(3)
    assert not bool(out[0].diagonal().any()) and bool(torch.isnan(out[0].triu(1)[0, 1]))
    grad = torch.autograd.grad(own(3).nan_to_num().tril().sum(), own.weight)[0]
    assert grad[:, 0].tolist() == [0.0, 3.0]
    with torch.autocast("cpu", dtype=BF16):
        assert m(2).dtype == BF16
    assert m(2, dtype=torch.float16).dtype == torch.float16 and m.double()(2).dtype == F64
    assert m(0, 4).shape == (3, 0, 4)


@pytest.mark.parametrize("p", [1.0, 2.0, INF])
def test_gradients_on_cpu(p):
    torch.manual_seed(0)
    grads = [torch.randn(30, 4), torch.randn(7).bfloat16(), torch.randn(3).double(), torch.empty(0)]
    flat = torch.cat([g.double().flatten() for g in grads])
    ref = flat.abs().max() if p == INF else flat.abs().sum() if p == 1 else flat.norm()
    norm = pkg.gradient_norm(grads, p)
    assert norm.dtype == F32 and torch.allclose(norm.double(), ref, rtol=1e-6)
    into = [torch.empty_like(g, dtype=F32) for g in grads]
    pkg.clip_gradients_(grads, 0.5, p, out=into)
    assert all(torch.allclose(o.double(), g.double() * 0.5 / ref, rtol=1e-5, atol=1e-9) for g, o in zip(grads, into))
    kept = [g.clone() for g in grads]
    pkg.clip_gradients_(grads, INF, p)
    assert all(torch.equal(a, b) for a, b in zip(grads, kept))
    pkg.clip_gradients_(grads, 0.5, p, norm=2 * norm)
    assert torch.allclose(grads[0], kept[0] * (0.25 / norm), rtol=1e-5)
    assert float(pkg.gradient_norm([], p)) == 0 and float(pkg.clip_gradients_([], 1.0, p)) == 0
    bad = [torch.tensor([1.0, math.nan]), torch.ones(2)]
    assert math.isnan(float(pkg.clip_gradients_(bad, 1.0, p))) and bool(torch.isnan(bad[1]).all())


def test_clip_grad_norm_as_torch_has_it():
    torch.manual_seed(0)
    nets = [torch.nn.Linear(5, 3), torch.nn.Linear(5, 3)]
    nets[1].load_state_dict(nets[0].state_dict())
    x = torch.randn(4, 5)
    for net in nets:
        (10 * net(x)).square().sum().backward()
    a = torch.nn.utils.clip_grad_norm_(nets[0].parameters(), 1.5)
    b = pkg.clip_grad_norm_(nets[1].parameters(), 1.5)
    assert torch.allclose(a, b)
    assert all(torch.allclose(p.grad, q.grad) for p, q in zip(nets[0].parameters(), nets[1].parameters()))
    nets[1].bias.grad[0] = INF
    with pytest.raises(RuntimeError, match="not finite"):
        pkg.clip_grad_norm_(nets[1].parameters(), 1.5, error_if_nonfinite=True)
    assert float(pkg.clip_grad_norm_(nets[1].weight, 1e9)) > 0
    assert float(pkg.clip_grad_norm_([torch.nn.Parameter(torch.ones(2))], 1.0)) == 0


@pytest.mark.parametrize("call,match", [
    (lambda: pkg.CudaGroupNorm(3, 8), "divide"),
    (lambda: pkg.CudaGroupNorm(2, 8, activation="tanh"), "activation"),
    (lambda: pkg.CudaGroupNorm(2, 8)(torch.zeros(2, 9)), "Expected"),
    (lambda: pkg.CudaGroupNorm(2, 8)(torch.zeros(8)), "Expected"),
    (lambda: pkg.CudaRelativeBias(0, 8), "positive"),
    (lambda: pkg.CudaRelativeBias(1, 8), "each side"),
    (lambda: pkg.CudaRelativeBias(32, 8, max_distance=8), "max_distance"),
    (lambda: pkg.CudaRelativeBias(4, 2, buckets=torch.zeros(4)), "far"),
    (lambda: pkg.CudaRelativeBias(4, 2)(-1), "negative"),
    (lambda: pkg.CudaRelativeBias(4, 2)(1, 2, offset=0, starts=torch.zeros(1, dtype=torch.int64)), "starts"),
    (lambda: pkg.clip_gradients_([torch.ones(2)], -1.0), "negative"),
    (lambda: pkg.clip_gradients_([torch.ones(2)], 1.0, 3.0), "norm_type"),
    (lambda: pkg.clip_gradients_([torch.ones(2)], 1.0, out=[]), "every gradient"),
    (lambda: pkg.gradient_norm([torch.ones(2).to_sparse()]), "dense"),
])
def test_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_example_with_clipping():
    """Runs with a limit; without one that is ever reached nothing changes."""
    from tests.test_example import _example

    run = lambda **kw: _example().train("cpu", steps=3, rows=512, batch=256, report=lambda s: None, **kw)  # noqa: E731
    assert run(clip=float("inf")) == run()
    assert all(map(torch.isfinite, map(torch.tensor, run(clip=0.1))))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("s", [1, 4096, 40_000])
@pytest.mark.parametrize("c,groups", [(1, 1), (60, 5), (77, 7), (520, 1), (960, 10), (1000, 10), (1280, 32), (4098, 2), (9000, 3),
                                      (20_001, 1), (30_000, 30), (1 << 20, 1)])
def test_group_norm_parameters_are_read_in_range(c, groups, s, dtype):
    """Every lane of a row's slabs, the last of which may be narrower than the others:
    the weight and bias have no channel behind the last."""
    forms = set()
    for n in (1, 300):
        for backward in (False, True):
            for x in (None, torch.empty(4)[1:], torch.empty(8, dtype=BF16)[1:]):
                plan = capi.group_norm_plan(n, s, c, groups, dtype, backward, x)
                assert plan["params_end"] == c, plan
                forms.add(plan["form"])
    assert 2 in forms if c >= 1000 and s > 4096 else True
    assert capi.group_norm_plan(0, s, c, groups)["params_end"] == 0


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("with_starts", [False, True])
@pytest.mark.parametrize("queries", [1, 4, None])
def test_relative_bias_compiles_once_for_all_lengths(queries, with_starts, train):
    """A decoding loop: a key more each time (queries None: as many queries as keys).  The
    first length and the lengths' symbol are the two graphs."""
    graphs = []

    def count(gm, inputs):
        graphs.append(gm)
        return gm.forward

    from torch._dynamo.backends.common import aot_autograd

    torch._dynamo.reset()
    starts = _meta(3, dtype=torch.int64) if with_starts else None
    buckets = _meta(9, dtype=torch.int32)

    def step(weight, k_len):
        q_len = k_len if queries is None else queries
        return _ops.relative_bias(weight, buckets, starts, q_len, k_len, k_len - q_len, True, F32) * 2

    compiled = torch.compile(step, backend=aot_autograd(fw_compiler=count, bw_compiler=lambda gm, _: gm.forward), fullgraph=True)
    for k_len in range(10, 30):
        weight = _meta(6, 4).requires_grad_(train)
        out = compiled(weight, k_len)
        assert out.shape[-2:] == (queries or k_len, k_len)
        if train:
            assert torch.autograd.grad(out.sum(), weight)[0].shape == (6, 4)
    torch._dynamo.reset()
    assert len(graphs) == 2


def test_relative_bias_compiles_with_symbolic_tables():
    """Every size a symbol, the table's rows and heads too."""
    torch._dynamo.reset()

    def step(weight, buckets, x):
        return _ops.relative_bias(weight, buckets, None, x.shape[0], x.shape[1], x.shape[1] - x.shape[0], False, F32).sum()

    compiled = torch.compile(step, backend="aot_eager", fullgraph=True, dynamic=True)
    for r, h, q, k in ((6, 4, 3, 5), (7, 5, 4, 8), (9, 2, 2, 3)):
        weight = _meta(r, h).requires_grad_()
        with torch._dynamo.config.patch(error_on_recompile=r > 6):
            (grad,) = torch.autograd.grad(compiled(weight, _meta(2 * r + 1, dtype=torch.int32), _meta(q, k)), weight)
        assert grad.shape == (r, h)
    torch._dynamo.reset()


def test_clip_grad_norm_takes_the_arguments_of_torch():
    """Called as torch's, with every argument by name and in its place."""
    import inspect

    theirs = list(inspect.signature(torch.nn.utils.clip_grad_norm_).parameters)
    assert list(inspect.signature(pkg.clip_grad_norm_).parameters)[:len(theirs)] == theirs
    p = torch.nn.Parameter(torch.ones(4))
    for foreach in (None, True, False):
        p.grad = torch.full((4,), 3.0)
        assert float(pkg.clip_grad_norm_([p], 1.5, 2.0, False, foreach)) == 6.0
        torch.testing.assert_close(p.grad, torch.full((4,), 0.75))
        assert float(pkg.clip_grad_norm_(p, max_norm=9.0, norm_type=2.0, error_if_nonfinite=True, foreach=foreach)) == pytest.approx(1.5)


@pytest.mark.parametrize("shape", [(0, 5, 12), (2, 0, 12), (0, 12)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda t: str(t)[6:])
def test_module_group_norm_without_rows_on_cpu(shape, dtype):
    """As on a device: parameters have gradients, of zeros."""
    m = pkg.CudaGroupNorm(3, 12, activation="silu")
    x = torch.empty(shape, dtype=dtype, requires_grad=True)
    y = m(x)
    assert y.shape == shape and y.dtype == dtype
    y.sum().backward()
    assert x.grad.shape == shape
    assert torch.equal(m.weight.grad, torch.zeros(12)) and torch.equal(m.bias.grad, torch.zeros(12))
    assert pkg.CudaGroupNorm(3, 12, affine=False)(x).shape == shape


def test_relative_bias_of_far_positions_on_cpu():
    """Positions beyond 2^60 count as 2^60, at either end of what 64 bits hold."""
    m = pkg.CudaRelativeBias(8, 2, max_distance=20, causal=True)
    starts = torch.tensor([2 ** 63 - 1, 2 ** 60, -2 ** 63, -2 ** 60])
    out = m(2, 3, starts=starts)
    past = m.weight[m.buckets[0].long()]
    assert torch.equal(out[:2], past[:, None, None].expand(2, 2, 2, 3))
    assert bool(torch.isneginf(out[2:]).all())


def test_relative_bias_starts_of_32_bits_on_cpu():
    m = pkg.CudaRelativeBias(8, 2, max_distance=20)
    starts = torch.tensor([5, 0, 90])
    assert torch.equal(m(4, 9, starts=starts.int()), m(4, 9, starts=starts))


@pytest.mark.parametrize("call,match", [
    (lambda g: pkg.clip_gradients_(g, 0.5, out=[torch.zeros(3, 4), torch.zeros(5)]), "shape"),
    (lambda g: pkg.clip_gradients_(g, 0.5, out=[torch.zeros(2, 3, 4), torch.zeros(4)]), "shape"),
    (lambda g: pkg.clip_gradients_(g, 0.5, out=[torch.zeros(1), torch.zeros(4)]), "shape"),
    (lambda g: pkg.clip_gradients_([*g, g[0]], 0.5), "share memory"),
    (lambda g: pkg.clip_gradients_([*g, g[0][:, :2]], 0.5), "share memory"),
    (lambda g: pkg.clip_gradients_([g[1], g[1].clone()], 0.5, out=[g[0][0], g[0][0]]), "share memory"),
])
def test_clipping_refusals_on_cpu(call, match):
    """As on a device; nothing is scaled."""
    grads = [torch.ones(3, 4), torch.ones(4)]
    with pytest.raises(ValueError, match=match):
        call(grads)
    assert all(bool((g == 1).all()) for g in grads)


def test_clipping_into_others_compiles_and_has_shapes():
    """On the CPU in one graph, and on meta tensors, which have no memory to share."""
    torch._dynamo.reset()
    grads = [torch.ones(3, 4), torch.ones(4)]
    want, got = ([torch.empty_like(g) for g in grads] for _ in range(2))
    norm = pkg.clip_gradients_(grads, 0.5, out=want)
    compiled = torch.compile(lambda g, o: pkg.clip_gradients_(g, 0.5, out=o), backend="eager", fullgraph=True)
    assert torch.equal(compiled(grads, got), norm) and all(map(torch.equal, got, want))
    torch._dynamo.reset()
    metas = [_meta(3, 4), _meta(4)]
    assert pkg.clip_gradients_(metas, 0.5, out=[_meta(3, 4), _meta(4)]).shape == ()

"""The operators around the embedding without a GPU: refusals of the C ABI,
FakeTensor contracts, autograd formulas (meta tensors), and the modules' CPU
path against 64-bit computations."""

from __future__ import annotations

import ctypes

import pytest
import torch

import piecewiselinearembeddings_optimized_amd as pkg
from piecewiselinearembeddings_optimized_amd import capi

_ops = torch.ops.rtdl_num_embeddings_cuda
F32, BF16 = torch.float32, torch.bfloat16
P = ctypes.c_void_p(256)


def test_c_abi_refuses_lookups():
    lib = capi.lib()

    def forward(tokens=P, size=8, offsets=None, weight=P, out=P, t=4, f=1, v=5, d=3, wt=0, ot=0):
        return lib.ple_lookup_launch(tokens, size, offsets, weight, out, t, f, v, d, 1.0, wt, ot, None)

    assert forward(t=0) == 0
    assert forward(size=2) == -4
    assert forward(v=0) == forward(d=0) == forward(t=-1) == forward(offsets=P, f=3) == -2
    assert forward(wt=7) == forward(ot=-1) == -3
    assert forward(tokens=None) == forward(weight=None) == forward(out=None) == -1
    assert forward(t=1 << 31) == forward(v=1 << 31) == forward(d=(1 << 20) + 1) == -5
    odd = ctypes.c_void_p(257)
    assert forward(tokens=odd) == forward(weight=odd) == forward(out=odd) == -8
    assert lib.ple_lookup_backward_launch(P, P, 8, None, None, 4, 1, 5, 3, -1, 1.0, 0, 0, None, 0, None) == -1
    assert lib.ple_lookup_backward_launch(P, P, 8, None, P, 4, 1, 5, 3, -1, 1.0, 0, 0, None, 0, None) == -6
    assert lib.ple_lookup_backward_workspace_bytes(0, 5, 3) == 0
    assert lib.ple_lookup_backward_workspace_bytes(4, 0, 3) == 0
    assert lib.ple_lookup_backward_workspace_bytes(1000, 50, 32) > 8000


def test_lookup_backward_grids():
    """Every launch of a gradient that a device can hold has fewer than 2^32 threads, however many rows are cleared."""
    most = 0
    for v in (1, 1000, 65_536, 1 << 20, 2_097_153, 4_194_303, 4_300_000, 6_300_000, 9_000_001, 1 << 24, 500_000_000, (1 << 31) - 2):
        for d in (1, 2, 7, 64, 1000, 4096, 8200, 8192, 12_288, 16_384, 100_000, 1 << 20):
            for t in (0, 1, 8192, 8193, 65_536, 3_000_000, (1 << 31) - 2):
                for g, w in ((F32, F32), (BF16, BF16), (BF16, F32)):
                    size = 4 if w == F32 else 2
                    fits = v * d * size + t * d * (4 if g == F32 else 2) < 288 << 30
                    try:
                        plan = capi.lookup_backward_plan(t, v, d, g, w)
                    except capi.PleError as e:
                        assert e.code == -5 and not fits, (t, v, d)
                        continue
                    assert plan["most_threads"] < 1 << 32
                    assert plan["clear_rows"] == max(1, 32768 // (d * size), -(-v // (1 << 21)))
                    assert plan["one_workgroup"] == (0 < t <= 8192)
                    assert plan["workspace_bytes"] == capi.lib().ple_lookup_backward_workspace_bytes(t, v, d)
                    if fits:
                        most = max(most, plan["most_threads"])
    assert most > 1 << 30
    assert capi.lookup_backward_plan(65_536, 131_072, 2048, BF16) | {"workspace_bytes": 0, "most_threads": 0} == {
        "one_workgroup": 0, "passes": 2, "digit_bits": 9, "sort_workgroups": 32, "sum_workgroups": 1024, "clear_rows": 8,
        "most_threads": 0, "workspace_bytes": 0}
    for bad in ((-1, 5, 3), (4, 0, 3), (4, 5, 0)):
        with pytest.raises(capi.PleError, match="shape"):
            capi.lookup_backward_plan(*bad)


def test_c_abi_refuses_norms():
    lib = capi.lib()

    def forward(n=4, d=8, branch=P, out=P, normed=P, stats=P, **kw):
        desc = capi.norm(F32, F32, 1, 1)
        for k, v in kw.items():
            setattr(desc, k, v)
        return lib.ple_residual_norm_launch(P, branch, ctypes.byref(desc), out, normed, stats, n, d, None)

    assert forward(n=0) == 0
    assert lib.ple_residual_norm_launch(P, P, None, P, P, P, 4, 8, None) == -1
    assert forward(n=-1) == forward(d=0) == -2
    assert forward(d=8193) == -5
    assert forward(param_dtype=9) == -3
    assert forward(stream_dtype=1) == -7                                     # a 16-bit stream of another type
    assert forward(post_norm=3) == forward(pre_norm=-1) == forward(gate_activation=3) == -7
    assert forward(post_norm=0, post_weight=256) == -7
    assert forward(gate=256, gate_rows=3) == forward(gate=256, gate_rows=0) == -2
    assert forward(branch=None, out=None) == -7                              # a post norm without a branch
    assert forward(branch=None, out=None, post_norm=0, residual_scale=0.5) == -7
    assert forward(out=None) == forward(normed=None) == forward(stats=None) == forward(pre_norm=0) == -1
    assert forward(branch=ctypes.c_void_p(258)) == forward(post_weight=257) == -8
    desc = capi.norm(F32, F32, 1, 1)
    grads = capi.NormGrads(gate=256)
    assert lib.ple_residual_norm_backward_launch(P, P, P, P, P, ctypes.byref(desc), ctypes.byref(grads), 4, 8, None, 0,
                                                 None) == -1                 # a gate's gradient without a gate


def test_c_abi_refuses_distillation():
    lib = capi.lib()

    def forward(z=P, size=8, loss=P, n=4, v=10, k=3, temperature=2.0, alpha=0.5, dtype=0, teacher=0):
        return lib.ple_distill_launch(z, P, P, size, None, None, loss, P, n, v, k, temperature, alpha, dtype, teacher, None,
                                      0, None)

    assert forward(n=0) == 0
    assert forward(n=-1) == forward(v=0) == forward(k=0) == -2
    assert forward(dtype=5) == forward(teacher=5) == -3
    assert forward(size=1) == -4
    assert forward(v=(1 << 30) + 1) == forward(k=(1 << 20) + 1) == forward(n=(1 << 24) + 1) == -5
    for t in (0.0, -1.0, 1e7, float("nan"), float("inf")):
        assert forward(temperature=t) == -7
    for a in (-0.1, 1.1, float("nan")):
        assert forward(alpha=a) == -7
    assert forward(z=None) == forward(loss=None) == -1
    assert forward(z=ctypes.c_void_p(258)) == -8
    assert forward(n=1, v=1 << 20) == -6                                     # split rows need a workspace
    assert lib.ple_distill_workspace_bytes(1, 1 << 20) > 0
    assert lib.ple_distill_workspace_bytes(4, 10) == 0


def _meta(*shape, dtype=F32):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_fake_shapes():
    out = _ops.lookup(_meta(3, 4, dtype=torch.int64), _meta(9, 6, dtype=BF16), None, 2.0, -1, F32)
    assert out.shape == (3, 4, 6) and out.dtype == F32
    dw = _ops.lookup_backward(out, _meta(3, 4, dtype=torch.int64), None, 9, 2.0, -1, BF16)
    assert dw.shape == (9, 6) and dw.dtype == BF16
    s, n, st = _ops.residual_norm(_meta(2, 5, 8), _meta(2, 5, 8, dtype=BF16), _meta(8), None, _meta(2, 8), _meta(8), None, 1, 2,
                                  0, 1.0, 1e-5, BF16)
    assert s.shape == n.shape == (2, 5, 8) and (s.dtype, n.dtype) == (F32, BF16) and st.shape == (10, 4)
    loss, stats = _ops.distillation_loss(_meta(7, 30), _meta(7, 4), _meta(7, 4, dtype=torch.int32), None, None, 1.0, 1.0)
    assert loss.shape == (7,) and stats.shape == (7, 8)
    with pytest.raises(RuntimeError, match="last dimension of tokens"):
        _ops.lookup(_meta(3, 4, dtype=torch.int64), _meta(9, 6), _meta(3, dtype=torch.int64), 1.0, -1, F32)
    with pytest.raises(RuntimeError, match="branch must have the shape"):
        _ops.residual_norm(_meta(2, 8), _meta(3, 8), None, None, None, None, None, 1, 1, 0, 1.0, 1e-5, F32)
    with pytest.raises(RuntimeError, match="temperature must be"):
        _ops.distillation_loss(_meta(7, 30), _meta(7, 4), _meta(7, 4, dtype=torch.int32), None, None, 0.0, 1.0)


def _recorded(op):
    """An operator's differentiable output on meta tensors, and what is differentiated."""
    if op == "lookup":
        wrt = [_meta(9, 6).requires_grad_()]
        return _ops.lookup(_meta(5, dtype=torch.int64), wrt[0], None, 2.0, 1, F32), wrt
    if op == "residual_norm":
        wrt = [_meta(4, 8).requires_grad_(), _meta(4, 8).requires_grad_(), *(_meta(8).requires_grad_() for _ in range(2)),
               _meta(2, 8).requires_grad_(), *(_meta(8).requires_grad_() for _ in range(2))]
        s, n, _ = _ops.residual_norm(*wrt, 2, 2, 1, 0.5, 1e-5, F32)
        return s + n, wrt
    wrt = [_meta(6, 20).requires_grad_()]
    return _ops.distillation_loss(wrt[0], _meta(6, 3), _meta(6, 3, dtype=torch.int64), _meta(6), _meta(6, dtype=torch.int64),
                                  2.0, 0.5)[0], wrt


OPS = ["lookup", "residual_norm", "distillation_loss"]


@pytest.mark.parametrize("op", OPS)
def test_autograd_formulas(op):
    out, wrt = _recorded(op)
    assert [g.shape for g in torch.autograd.grad(out.sum(), wrt)] == [t.shape for t in wrt]


def test_statistics_are_not_differentiable():
    r, b, w = _meta(4, 8).requires_grad_(), _meta(4, 8).requires_grad_(), _meta(8).requires_grad_()

    def norm(branch, post, pre):
        out = _ops.residual_norm(r, branch, w if post else None, None, None, w if pre else None, None, post, pre, 0, 1.0, 1e-5, F32)
        return [t.requires_grad for t in out]

    assert norm(b, 1, 2) == [True, True, False]
    assert norm(b, 1, 0) == [True, False, False]            # no norm before a block: an empty output
    assert norm(None, 0, 2) == [False, True, False]         # no branch: an empty stream
    loss, stats = _ops.distillation_loss(_meta(6, 20).requires_grad_(), _meta(6, 3), _meta(6, 3, dtype=torch.int64), None, None,
                                         2.0, 0.5)
    assert loss.requires_grad and not stats.requires_grad


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
            if op == "lookup":
                _ops.lookup(_meta(5, dtype=torch.int64), dual, None, 2.0, 1, F32)
            elif op == "residual_norm":
                _ops.residual_norm(dual, *wrt[1:], 2, 2, 1, 0.5, 1e-5, F32)
            else:
                _ops.distillation_loss(dual, _meta(6, 3), _meta(6, 3, dtype=torch.int64), None, None, 2.0, 0.5)


def test_module_lookup_on_cpu():
    torch.manual_seed(0)
    m = pkg.CudaCategoricalEmbeddings([3, 5], 4, scale=2.0)
    t = torch.tensor([[0, 4], [-1, 0], [2, 5]])
    out = m(t)
    assert torch.equal(out[0, 0], 2 * m.weight[0]) and torch.equal(out[0, 1], 2 * m.weight[7])
    assert not bool(out[1, 0].any()) and bool(torch.isnan(out[2, 1]).all())
    g = torch.autograd.grad(out[:2].sum(), m.weight)[0]
    assert torch.equal(g[:, 0], torch.tensor([2.0, 0, 0, 2, 0, 0, 0, 2]))
    assert m.get_output_shape() == (2, 4)
    e = pkg.CudaTokenEmbeddings(6, 3, padding_idx=1)
    assert torch.equal(e(torch.tensor([1])), e.weight[1:2])
    assert torch.equal(torch.autograd.grad(e(torch.tensor([1, 2])).sum(), e.weight)[0][:3, 0], torch.tensor([0.0, 0, 1]))
    with torch.autocast("cpu", dtype=BF16):
        assert e(torch.tensor([0])).dtype == BF16


def test_module_norm_on_cpu():
    torch.manual_seed(0)
    m = pkg.CudaResidualNorm(16, post_norm="layer", pre_norm="rms", bias=True, residual_scale=0.5)
    r, b, g = torch.randn(2, 3, 16), torch.randn(2, 3, 16), torch.randn(2, 1, 16)
    s, n = m(r, b, g)
    ref = 0.5 * r.double() + g.double() * torch.nn.functional.layer_norm(b.double(), (16,), eps=1e-5)
    torch.testing.assert_close(s.double(), ref, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(n.double(), ref * (ref.square().mean(-1, keepdim=True) + 1e-5).rsqrt(), rtol=1e-5, atol=1e-5)
    assert m(r)[0] is r
    end = pkg.CudaResidualNorm(16, pre_norm=None, gate="learned", gate_init=0.0, gate_activation="tanh")
    s, n = end(r, b)
    assert s is n and torch.equal(s, r)
    assert [k for k, _ in end.named_parameters()] == ["gate"]


def test_module_loss_on_cpu():
    torch.manual_seed(0)
    z, t, c = torch.randn(4, 10), torch.randn(4, 3), torch.tensor([[0, 1, 2], [3, -1, 4], [-1, -1, -1], [9, 8, 7]])
    loss = pkg.CudaDistillationLoss(2.0, 1.0, "none")(z, t, c)
    for i, keep in enumerate(([0, 1, 2], [0, 2], [], [0, 1, 2])):
        want = 0.0
        if keep:
            lp = torch.log_softmax(t[i, keep].double() / 2, 0)
            want = 4 * float((lp.exp() * (lp - torch.log_softmax(z[i].double() / 2, 0)[c[i, keep]])).sum())
        assert abs(float(loss[i]) - want) < 1e-5
    labels = torch.tensor([1, -100, 10, 3])
    hard = pkg.CudaDistillationLoss(2.0, 0.0, "none")(z, t, c, labels=labels)
    assert hard[1] == 0 and torch.isnan(hard[2])
    assert abs(float(hard[3]) + float(torch.log_softmax(z[3], 0)[3])) < 1e-5
    # the whole teacher with its own lse is the plain divergence, and splits off nothing
    full = torch.randn(2, 10)
    a = pkg.CudaDistillationLoss(1.5, 1.0, "none")(z[:2], full, torch.arange(10).expand(2, 10),
                                                   torch.logsumexp(full / 1.5, -1))
    b = pkg.CudaDistillationLoss(1.5, 1.0, "none")(z[:2], full, torch.arange(10).expand(2, 10))
    torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)


def test_module_loss_outside_mass_below_32_bits():
    """A student whose mass outside the teacher's classes has no number in 32 bits."""
    gen = torch.Generator().manual_seed(3)
    z, t = torch.randn(5, 20, generator=gen), torch.randn(5, 4, generator=gen)
    c = torch.arange(4).expand(5, 4).contiguous()
    z[:, 4:] -= 300
    z.requires_grad_()
    lse = torch.logsumexp(t, -1) + 0.3
    got = pkg.CudaDistillationLoss(1.0, 1.0, "sum")(z, t, c, lse)
    zd = z.detach().double().requires_grad_()
    log_q, log_p = torch.log_softmax(zd, -1), t.double() - lse.double()[:, None]
    rho = 1 - log_p.exp().sum(-1)
    want = ((log_p.exp() * (log_p - log_q[:, :4])).sum(-1) + rho * (rho.log() - torch.logsumexp(log_q[:, 4:], -1))).sum()
    torch.testing.assert_close(got.double(), want, rtol=1e-5, atol=0)
    torch.testing.assert_close(torch.autograd.grad(got, z)[0].double(), torch.autograd.grad(want, zd)[0], rtol=1e-4, atol=1e-5)


def test_module_loss_teacher_has_no_gradient():
    z, t, lse = torch.randn(3, 6).requires_grad_(), torch.randn(3, 2).requires_grad_(), torch.ones(3).requires_grad_()
    loss = pkg.CudaDistillationLoss(2.0)(z, t, torch.arange(2).repeat(3, 1), lse)
    grads = torch.autograd.grad(loss, (z, t, lse), allow_unused=True)
    assert grads[0] is not None and grads[1:] == (None, None)


@pytest.mark.parametrize("tail", [False, True])
def test_module_loss_of_classes_and_labels_beyond(tail):
    """A class or label beyond the logits': the row's loss and its whole gradient are NaN, no other row's."""
    gen = torch.Generator().manual_seed(5)
    z, t, c = torch.randn(6, 7, generator=gen), torch.randn(6, 3, generator=gen), torch.arange(3).repeat(6, 1)
    c[1, 2] = 7
    c[4, 0], z[4] = 9, -torch.inf                   # (a row without any class left has no loss)
    label = torch.tensor([0, 1, 7, -100, 2, 6])
    z.requires_grad_()
    for alpha, bad in ((0.5, [1, 2]), (1.0, [1]), (0.0, [2])):
        loss = pkg.CudaDistillationLoss(2.0, alpha, "none")(z, t, c, torch.full((6,), 2.0) if tail else None, label)
        grad = torch.autograd.grad(loss.sum(), z)[0]
        want = torch.zeros(6, dtype=torch.bool)
        want[bad] = True
        assert torch.equal(torch.isnan(loss), want)
        assert torch.equal(torch.isnan(grad).all(1), want) and torch.equal(torch.isnan(grad).any(1), want)
        assert loss[4] == 0 and not bool(grad[4].any())


@pytest.mark.parametrize("labels", [False, True])
def test_module_loss_without_an_outside(labels):
    """Rows whose classes beside the teacher's are all masked: no outside, and a finite gradient."""
    gen = torch.Generator().manual_seed(4)
    z, t = torch.randn(4, 9, generator=gen), torch.randn(4, 5, generator=gen)
    c = torch.arange(5).expand(4, 5).contiguous()
    z[:2, 5:] = -torch.inf                          # every class that is left is the teacher's
    z[2, 5:] = torch.finfo(F32).min
    label = torch.tensor([0, 3, 4, 7]) if labels else None
    lse = torch.logsumexp(t / 2, -1) + 0.3
    z.requires_grad_()
    got = pkg.CudaDistillationLoss(2.0, 0.7, "none")(z, t, c, lse, label)
    zd = z.detach().double().requires_grad_()
    log_q, log_p = torch.log_softmax(zd / 2, -1)[:, :5], t.double() / 2 - lse.double()[:, None]
    kd = (log_p.exp() * (log_p - log_q)).sum(-1)
    rho = 1 - log_p[3].exp().sum()
    rest = rho * (rho.log() - torch.logsumexp(torch.log_softmax(zd[3] / 2, -1)[5:], -1))
    want = 0.7 * 4 * (kd + torch.cat([torch.zeros(3, dtype=torch.float64), rest[None]]))
    if labels:
        want = want - 0.3 * torch.log_softmax(zd, -1)[torch.arange(4), label]
    torch.testing.assert_close(got.double(), want, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(torch.autograd.grad(got.sum(), z)[0].double(), torch.autograd.grad(want.sum(), zd)[0],
                               rtol=1e-4, atol=1e-6)


def test_modules_in_64_bits_on_cpu():
    """float64 inputs are computed in 64 bits: differences of 1e-5 give the gradient to 1e-8."""
    torch.manual_seed(6)
    F64 = torch.float64
    e = pkg.CudaTokenEmbeddings(5, 3, scale=1 / 3).double()
    assert torch.equal(e(torch.tensor([2])), e.weight[2:3] * (1 / 3))
    m = pkg.CudaResidualNorm(6, post_norm="layer", pre_norm="rms", bias=True, gate="learned", gate_activation="tanh").double()
    r, b = torch.randn(4, 6, dtype=F64), torch.randn(4, 6, dtype=F64)
    s, n = m(r, b)
    ref = r + torch.tanh(m.gate) * torch.nn.functional.layer_norm(b, (6,), eps=1e-5)
    assert s.dtype == n.dtype == F64
    torch.testing.assert_close(s, ref, rtol=1e-13, atol=1e-13)
    torch.testing.assert_close(n, ref * (ref.square().mean(-1, keepdim=True) + 1e-5).rsqrt(), rtol=1e-13, atol=1e-13)
    z, t, c = torch.randn(3, 8, dtype=F64).requires_grad_(), torch.randn(3, 4, dtype=F64), torch.arange(4).repeat(3, 1)
    loss = pkg.CudaDistillationLoss(2.0, 0.6)
    value = lambda z: loss(z, t, c, torch.logsumexp(t / 2, -1) + 0.2, torch.tensor([1, 5, -1]))  # noqa: E731
    assert value(z).dtype == F64
    step = torch.randn_like(z)
    slope = (value(z + 1e-5 * step) - value(z - 1e-5 * step)) / 2e-5
    assert abs(float(slope - (torch.autograd.grad(value(z), z)[0] * step).sum())) < 1e-8


@pytest.mark.parametrize("call,match", [
    (lambda: pkg.CudaTokenEmbeddings(0, 3), "positive"),
    (lambda: pkg.CudaTokenEmbeddings(4, 3, padding_idx=4), "padding_idx"),
    (lambda: pkg.CudaCategoricalEmbeddings([], 3), "cardinalities"),
    (lambda: pkg.CudaCategoricalEmbeddings([3, 0], 3), "cardinalities"),
    (lambda: pkg.CudaCategoricalEmbeddings([3, 4], 3)(torch.zeros(5, 3, dtype=torch.int64)), "Expected 2"),
    (lambda: pkg.CudaResidualNorm(9000), "between 1 and"),
    (lambda: pkg.CudaResidualNorm(8, post_norm="batch"), "norms must be"),
    (lambda: pkg.CudaResidualNorm(8, gate="row"), "gate must be"),
    (lambda: pkg.CudaResidualNorm(8, gate_activation="relu"), "gate_activation"),
    (lambda: pkg.CudaResidualNorm(8)(torch.zeros(2, 7)), "rows of 8"),
    (lambda: pkg.CudaResidualNorm(8)(torch.zeros(2, 8), gate=torch.zeros(8)), "needs a branch"),
    (lambda: pkg.CudaResidualNorm(8)(torch.zeros(2, 3, 8), torch.zeros(2, 3, 8), torch.zeros(3, 8)), "broadcast"),
    (lambda: pkg.CudaResidualNorm(8, gate="learned")(torch.zeros(2, 8), torch.zeros(2, 8), torch.zeros(8)), "learned gate"),
    (lambda: pkg.CudaDistillationLoss(0.0), "temperature"),
    (lambda: pkg.CudaDistillationLoss(alpha=2.0), "alpha"),
    (lambda: pkg.CudaDistillationLoss(reduction="max"), "reduction"),
    (lambda: pkg.CudaDistillationLoss()(torch.zeros(3, 5), torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.int64)), "fit"),
])
def test_module_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()

"""Distillation loss and its gradient on the GPU against a 64-bit computation.

Tolerances.  With u = z / T every exponential's argument is rounded in 32 bits,
so a probability is off by about 2^-24 * (|u - max| + |log V| + 8) of itself;
below, e = 2^-24 * (40 + the largest finite |u - max| of the row) bounds it with
some room.  A loss adds the terms' sizes, a gradient's element is e of each term
it is made of, plus half a unit of the stored type.
"""

from __future__ import annotations

import math
import time

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
INF = float("inf")


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available(), "HIP device required"
    import piecewiselinearembeddings_optimized_amd  # noqa: F401  (registers the ops)

    return torch.ops.rtdl_num_embeddings_cuda


def _inputs(n, v, k, dtype=F32, tail=False, labels=True, seed=0, teacher=F32, repeat=False):
    gen = torch.Generator().manual_seed(seed + 7 * n + v)
    classes = torch.stack([torch.randperm(v, generator=gen)[:k] for _ in range(n)]) if not repeat else \
        torch.randint(0, v, (n, k), generator=gen)
    t = (3 * torch.randn(n, classes.shape[1], generator=gen)).sort(-1, descending=True).values.to(teacher)
    z = (2 * torch.randn(n, v, generator=gen)).scatter_add(1, classes, 0.7 * t.float()).to(dtype)
    return {"z": z, "t": t, "c": classes,
            "lse": torch.logsumexp(t.float(), -1) + 0.5 * torch.rand(n, generator=gen) if tail else None,
            "labels": torch.randint(0, v, (n,), generator=gen) if labels else None,
            "g": torch.randn(n, generator=gen)}


def _run(ops, x, temperature, alpha):
    dev = {k: None if v is None else v.to(DEV) for k, v in x.items()}
    loss, stats = ops.distillation_loss(dev["z"], dev["t"], dev["c"], dev["lse"], dev["labels"], temperature, alpha)
    dz = ops.distillation_loss_backward(dev["g"], dev["z"], dev["t"], dev["c"], dev["labels"], stats, temperature, alpha)
    return loss.cpu(), dz.cpu()


def _reference(x, temperature, alpha):
    """Loss, gradient, and the sizes of the terms they are made of, row by row in 64 bits."""
    n, v = x["z"].shape
    loss, loss_size = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
    dz, dz_size = torch.zeros(n, v, dtype=torch.float64), torch.zeros(n, v, dtype=torch.float64)
    eps = torch.zeros(n, dtype=torch.float64)
    for i in range(n):
        z = x["z"][i].double()
        if bool(torch.isneginf(z).all()):
            continue
        u = z / temperature
        log_q, log_1 = torch.log_softmax(u, 0), torch.log_softmax(z, 0)
        fin = torch.isfinite(z)
        eps[i] = 2.0 ** -24 * (40 + float((z[fin].max() - z[fin].min()).clamp_max(100)) * max(1.0, 1 / temperature))
        g = x["g"][i].double()
        here = x["c"][i] >= 0
        c, t = x["c"][i][here].long(), x["t"][i][here].double() / temperature
        if bool((c >= v).any()):
            loss[i] = float("nan")
            dz[i] = float("nan")
            continue
        if len(c) and alpha > 0 and (x["lse"] is not None or not bool(torch.isneginf(t).all())):
            lse = x["lse"][i].double() if x["lse"] is not None else torch.logsumexp(t, 0)
            lp = t - lse
            p = lp.exp()
            some = p > 0
            kd = (p[some] * (lp[some] - log_q[c[some]])).sum()
            size = (p[some] * (lp[some].abs() + log_q[c[some]].abs() + 1)).sum()
            named = torch.zeros(v, dtype=torch.bool)
            named[c] = True
            target = torch.zeros(v, dtype=torch.float64).index_add_(0, c, p)
            mass = p.sum()
            grad = log_q.exp() * mass - target
            gsize = log_q.exp() * mass + target
            if x["lse"] is not None:
                rho = (1 - mass).clamp_min(0)
                rest = log_q[~named].exp().sum()
                if rho > 0 and rest > 0:
                    kd = kd + rho * (rho.log() - rest.log())
                    size = size + rho * (rho.log().abs() + rest.log().abs() + 1) + rho.log().abs() + rest.log().abs()
                    grad = grad + rho * torch.where(named, log_q.exp(), log_q.exp() * (1 - 1 / rest))
                    # (rho is a difference from 1: off by some 2^-24, whatever its size)
                    gsize = gsize + log_q.exp() * (rho + 1) + torch.where(named, 0.0, log_q.exp() / rest) * (rho + 1)
            loss[i] += alpha * temperature ** 2 * kd
            loss_size[i] += alpha * temperature ** 2 * size
            dz[i] += g * alpha * temperature * grad
            dz_size[i] += abs(g) * alpha * temperature * gsize
        if x["labels"] is not None and alpha < 1:
            label = int(x["labels"][i])
            if label >= v:
                loss[i] = float("nan")
                dz[i] = float("nan")
            elif label >= 0:
                loss[i] -= (1 - alpha) * log_1[label]
                loss_size[i] += (1 - alpha) * (log_1[label].abs() + 1)
                hit = torch.zeros(v, dtype=torch.float64)
                hit[label] = 1
                dz[i] += g * (1 - alpha) * (log_1.exp() - hit)
                dz_size[i] += abs(g) * (1 - alpha) * (log_1.exp() + hit)
    return loss, loss_size, dz, dz_size, eps


def _check(ops, x, temperature=2.0, alpha=0.6):
    loss, dz = _run(ops, x, temperature, alpha)
    dtype = x["z"].dtype
    assert loss.dtype == F32 and dz.dtype == dtype
    ref, size, rdz, dsize, eps = _reference(x, temperature, alpha)
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(loss), nan)
    same = torch.isinf(ref) & (loss.double() == ref)
    off = (loss.double() - ref).abs()
    assert bool((nan | same | (off <= eps * size + 1e-30)).all()), float((off / (eps * size))[~nan & ~same].max())
    dz = dz.double()
    assert torch.equal(torch.isnan(dz), torch.isnan(rdz))
    bound = eps[:, None] * dsize + UNIT[dtype] * rdz.abs() + (2.0 ** -24 if dtype == F16 else 1e-37)
    ok = torch.isnan(rdz) | ((dz - rdz).abs() <= bound)
    assert bool(ok.all()), float(((dz - rdz).abs() / bound)[~torch.isnan(rdz)].max())


SHAPES = [(1, 1, 1), (3, 2, 2), (5, 7, 3), (70, 8, 8), (33, 64, 10), (9, 65, 64), (300, 100, 5), (10, 500, 20),
          (6, 2048, 32), (5, 2049, 300), (4, 5003, 64), (2, 10_240, 100), (1, 20_001, 17), (3, 50_257, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("n,v,k", SHAPES)
@pytest.mark.parametrize("tail", [False, True], ids=["top", "tail"])
def test_shapes(ops, n, v, k, dtype, tail):
    _check(ops, _inputs(n, v, k, dtype, tail))
    _check(ops, _inputs(n, v, k, dtype, tail, labels=False), temperature=1.0, alpha=1.0)


@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0, 10.0])
@pytest.mark.parametrize("alpha", [0.0, 0.3, 1.0])
@pytest.mark.parametrize("v", [30, 3001])
def test_temperatures_and_weights(ops, temperature, alpha, v):
    for tail in (False, True):
        for labels in (False, True):
            _check(ops, _inputs(12, v, 9, tail=tail, labels=labels), temperature, alpha)


@pytest.mark.parametrize("teacher", [F32, BF16, F16], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("wide", [False, True], ids=["i32", "i64"])
def test_teacher_types(ops, teacher, wide):
    x = _inputs(20, 333, 12, BF16, True, teacher=teacher)
    _check(ops, x if wide else dict(x, c=x["c"].int()))


@pytest.mark.parametrize("v", [6, 90, 3000, 9001])
@pytest.mark.parametrize("tail", [False, True], ids=["top", "tail"])
def test_absent_classes_labels_and_repeats(ops, v, tail):
    """Padding entries, rows without any, ignored labels, classes that occur twice."""
    x = _inputs(40, v, 24, tail=tail, repeat=True)
    gen = torch.Generator().manual_seed(v)
    x["c"][torch.rand(40, 24, generator=gen) < 0.3] = -1
    x["c"][3] = -7
    x["labels"][torch.rand(40, generator=gen) < 0.4] = -100
    x["c"][5], x["labels"][5] = -1, -100
    x["c"][8] = x["labels"][8]                      # one class 24 times, the label's too
    loss, dz = _run(ops, x, 2.0, 0.6)
    assert loss[5] == 0 and not bool(dz[5].any())
    if tail:                                        # (a teacher's mass above 1 has no rest)
        x["lse"] = torch.logsumexp(torch.where(x["c"] >= 0, x["t"] / 2, -INF), -1).nan_to_num(neginf=0.0) + 0.1
    _check(ops, x)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("v", [50, 700, 9000])
def test_masked_classes(ops, v, dtype):
    """-inf and the type's lowest value in the logits, and a row of nothing else."""
    x = _inputs(24, v, 8, dtype, True)
    low = torch.finfo(dtype).min
    masked = torch.rand(24, v, generator=torch.Generator().manual_seed(v)) < 0.3
    masked.scatter_(1, x["c"], False)
    masked.scatter_(1, x["labels"][:, None], False)
    x["z"][:12][masked[:12]] = -INF
    x["z"][12:][masked[12:]] = low
    x["z"][4] = -INF                                # nothing left
    x["z"][6] = low                                 # uniform
    x["z"][7] = -INF
    x["z"][7, int(x["labels"][7])] = 1.0            # one class: the teacher's others are impossible
    loss, dz = _run(ops, x, 2.0, 0.6)
    assert loss[4] == 0 and not bool(dz[4].any())
    assert loss[7] == INF and not bool(torch.isnan(dz[7]).any())
    keep = [i for i in range(24) if i != 7]
    _check(ops, {k: t[keep] for k, t in x.items()})


@pytest.mark.parametrize("dtype", [F32, BF16], ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("v", [14, 90, 3000, 40_000])
@pytest.mark.parametrize("temperature", [1.0, 1.5, 2.0])
def test_outside_mass_below_32_bits(ops, v, dtype, temperature):
    """A student that is sure of the teacher's classes: the mass outside them has no
    number in 32 bits, its logarithm and the outside classes' shares of it do."""
    x = _inputs(6, v, 8, F32, True)
    near = torch.zeros(6, v).scatter_(1, x["c"], 1.0)
    x["z"] = (x["z"] - 300 * (1 - near)).to(dtype)
    x["lse"] = torch.logsumexp(x["t"] / temperature, -1) + 0.3
    loss, _ = _run(ops, x, temperature, 0.6)
    assert bool((loss > 10).all())
    _check(ops, x, temperature)
    _check(ops, dict(x, labels=None), temperature, 1.0)


@pytest.mark.parametrize("v", [9, 70, 3000, 9000])
@pytest.mark.parametrize("temperature", [1.0, 1.5, 2.0])
def test_rows_without_an_outside(ops, v, temperature):
    """All classes beside the teacher's are masked: no outside, as on the CPU."""
    from piecewiselinearembeddings_optimized_amd import CudaDistillationLoss

    x = _inputs(6, v, 5, tail=True)
    named = torch.zeros(6, v, dtype=torch.bool).scatter_(1, x["c"], True)
    x["z"][:3][~named[:3]] = -INF
    x["z"][3][~named[3]] = torch.finfo(F32).min
    x["labels"] = x["c"][:, 2].clone()
    x["lse"] = torch.logsumexp(x["t"] / temperature, -1) + 0.3
    _check(ops, x, temperature)
    m = CudaDistillationLoss(temperature, 0.6, "sum")
    grads = []
    for dev in ("cpu", DEV):
        z = x["z"].to(dev).requires_grad_()
        grads.append(torch.autograd.grad(m(z, *(x[k].to(dev) for k in ("t", "c", "lse", "labels"))), z)[0].cpu())
    assert bool(torch.isfinite(grads[0]).all())
    torch.testing.assert_close(grads[1], grads[0], rtol=1e-4, atol=1e-5)


def test_large_and_non_finite_logits(ops):
    x = _inputs(10, 400, 8, tail=True)
    x["z"][0] *= 1e4
    x["z"][1] += 1e6
    x["z"][2, 7] = INF
    x["z"][3, 9] = float("nan")
    loss, dz = _run(ops, x, 2.0, 0.6)
    assert torch.isnan(loss[2:4]).all() and torch.isnan(dz[2:4]).any(1).all()
    assert bool(torch.isfinite(loss[[0, 1, 4, 5, 6, 7, 8, 9]]).all())
    keep = [4, 5, 6, 7, 8, 9]
    _check(ops, {k: t[keep] for k, t in x.items()})


def test_teacher_without_mass(ops):
    """Teacher logits of -inf: no probability; a row of them has no teacher."""
    x = _inputs(6, 40, 5, labels=True)
    x["t"][0, 2:] = -INF
    x["t"][1] = -INF
    _check(ops, x)


def test_classes_and_labels_beyond(ops):
    x = _inputs(12, 300, 6)
    x["c"][2, 3] = 300
    x["c"][4, 0] = 1 << 40
    x["labels"][7] = 300
    loss, dz = _run(ops, x, 2.0, 0.6)
    bad = torch.zeros(12, dtype=torch.bool)
    bad[[2, 4, 7]] = True
    assert torch.equal(torch.isnan(loss), bad) and torch.equal(torch.isnan(dz).all(1), bad)
    assert torch.equal(torch.isnan(dz).any(1), bad)
    _check(ops, {k: None if t is None else t[~bad] for k, t in x.items()})


@pytest.mark.parametrize("alpha", [0.0, 0.5, 1.0])
def test_classes_and_labels_beyond_as_on_the_cpu(ops, alpha):
    from piecewiselinearembeddings_optimized_amd import CudaDistillationLoss

    x = _inputs(9, 40, 4, tail=True)
    x["c"][1, 2] = 40
    x["c"][4, 0], x["z"][4] = 90, -INF              # nothing left: no loss
    x["labels"][2], x["labels"][6] = 40, -100
    m = CudaDistillationLoss(2.0, alpha, "none")
    out = []
    for dev in ("cpu", DEV):
        z = x["z"].to(dev).requires_grad_()
        loss = m(z, *(x[k].to(dev) for k in ("t", "c", "lse", "labels")))
        out.append((loss.detach().cpu(), torch.autograd.grad(loss.sum(), z)[0].cpu()))
    for a, b in zip(*out):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5, equal_nan=True)


def test_more_entries_than_classes(ops):
    _check(ops, _inputs(4, 5, 200, repeat=True))
    _check(ops, _inputs(2, 3000, 2500, tail=True))


@pytest.mark.parametrize("k", [80, 81, 97, 193, 576, 577, 3000])
@pytest.mark.parametrize("v", [40, 500, 3000, 9000, 40_000, 300_000])
@pytest.mark.parametrize("tail", [False, True], ids=["top", "tail"])
def test_many_entries_with_repeats(ops, v, k, tail):
    """Rows whose entries repeat classes, some, none or all, beside each other.  A class of
    m entries adds up m probabilities one after another: off by up to m 2^-24 of their sum."""
    n = 5
    x = _inputs(n, v, k, tail=tail, repeat=True)
    gen = torch.Generator().manual_seed(k)
    x["c"][0, :k // 2] = x["c"][0, 0]               # one class for half of the entries
    x["c"][1, 7:] = -1                              # few entries
    x["c"][2] = torch.arange(k) if k <= v else torch.arange(k) % v
    x["c"][3] = x["labels"][3]                      # one class in all, the label's too
    x["c"][4][torch.rand(k, generator=gen) < 0.5] = -3
    if tail:
        x["lse"] = torch.logsumexp(torch.where(x["c"] >= 0, x["t"] / 2, -INF), -1) + 0.4
    loss, dz = _run(ops, x, 2.0, 0.6)
    ref, size, rdz, dsize, eps = _reference(x, 2.0, 0.6)
    most = torch.stack([c[c >= 0].bincount().max() for c in x["c"]])
    eps = eps + 2.0 ** -24 * (most + k / 8)         # (and the row's sums of a lane's entries)
    assert bool(((loss.double() - ref).abs() <= eps * size).all()), ((loss.double() - ref).abs() / (eps * size))
    assert bool(((dz.double() - rdz).abs() <= eps[:, None] * dsize + UNIT[F32] * rdz.abs() + 1e-37).all())
    again = _run(ops, x, 2.0, 0.6)
    assert torch.equal(again[0], loss) and torch.equal(again[1], dz)


def test_repeats_take_no_square_of_the_entries(ops):
    """131072 entries a row, all of them twice: 2^34 comparisons if each looked for its class."""
    n, v, k = 4, 70_000, 1 << 17
    gen = torch.Generator().manual_seed(0)
    half = torch.stack([torch.randperm(v, generator=gen)[:k // 2] for _ in range(n)])
    x = {"z": torch.randn(n, v, generator=gen), "t": torch.randn(n, k, generator=gen), "c": torch.cat([half, half], 1),
         "lse": None, "labels": None, "g": torch.ones(n)}
    x["lse"] = torch.logsumexp(x["t"], -1) + 0.2
    _run(ops, {key: None if t is None else t[:, :4].contiguous() if key in "tc" else t for key, t in x.items()}, 1.0, 1.0)
    start = time.monotonic()
    loss, dz = _run(ops, x, 1.0, 1.0)
    assert time.monotonic() - start < 2.0
    # each class once, with the sum of its two probabilities
    p = torch.softmax(x["t"].double(), -1) * math.exp(-0.2)
    target = torch.zeros(n, v, dtype=torch.float64).scatter_add_(1, x["c"], p)
    log_q = torch.log_softmax(x["z"].double(), -1)
    named = torch.zeros(n, v, dtype=torch.bool).scatter_(1, x["c"], True)
    rho = 1 - math.exp(-0.2)
    rest = torch.where(named, 0.0, log_q.exp()).sum(-1, keepdim=True)
    want = (p * (p.log() - log_q.gather(1, x["c"]))).sum(-1) + rho * (math.log(rho) - rest.log())[:, 0]
    grad = log_q.exp() - target - torch.where(named, 0.0, rho * log_q.exp() / rest)
    # (a lane's 512 entries and the sums of 2^17 probabilities: some 2^-24 * 600 of the terms)
    torch.testing.assert_close(loss.double(), want, rtol=4e-5 * 12, atol=0)
    assert bool(((dz.double() - grad).abs() <= 4e-5 * (target + log_q.exp() * (1 + rho / rest))).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [33, 1001, 7000])
def test_unaligned_rows(ops, dtype, v):
    """Logits and their gradient at addresses a different way into 16 bytes."""
    x = _inputs(5, v, 6, dtype, True)
    loss, dz = _run(ops, x, 2.0, 0.6)
    base = torch.zeros(5 * v + 1, dtype=dtype, device=DEV)
    base[1:] = x["z"].to(DEV).reshape(-1)
    dev = {k: t.to(DEV) for k, t in x.items()}
    z = base[1:].view(5, v)
    l2, stats = ops.distillation_loss(z, dev["t"], dev["c"], dev["lse"], dev["labels"], 2.0, 0.6)
    d2 = ops.distillation_loss_backward(dev["g"], z, dev["t"], dev["c"], dev["labels"], stats, 2.0, 0.6)
    torch.testing.assert_close(l2.cpu(), loss, rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(d2.cpu(), dz, rtol=2e-2 if dtype == BF16 else 1e-4, atol=1e-6)


def test_very_many_classes(ops):
    """More classes than one workgroup has bits for."""
    _check(ops, _inputs(2, 600_011, 40, BF16, True))


def test_more_rows_than_one_grid(ops):
    """2^24 rows by workgroups: 2^32 threads, in two launches."""
    n, v = 1 << 24, 4100
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip("needs 150 GB of device memory")
    z = torch.zeros(n, v, dtype=F16, device=DEV)
    c = (torch.arange(n, device=DEV, dtype=torch.int32) % v).reshape(n, 1)
    at = torch.tensor([0, 77, (1 << 23) - 1, 1 << 23, (1 << 23) + 5, n - 1], device=DEV)
    z[at, c[at, 0].long()] = 5.0
    loss, stats = ops.distillation_loss(z, torch.ones(n, 1, device=DEV), c, None, None, 1.0, 1.0)
    del z
    far = torch.ones(n, dtype=torch.bool, device=DEV)
    far[at] = False
    torch.testing.assert_close(loss[far], torch.full_like(loss[far], math.log(v)), rtol=1e-5, atol=0)
    torch.testing.assert_close(loss[at].cpu(), torch.full((6,), math.log(v - 1 + math.exp(5.0)) - 5.0), rtol=1e-5, atol=0)
    assert stats.shape == (n, 8)
    torch.cuda.empty_cache()                        # (half of the device)


def test_empty(ops):
    x = _inputs(1, 20, 3)
    x = {k: None if t is None else t[:0] for k, t in x.items()}
    loss, dz = _run(ops, x, 2.0, 0.5)
    assert loss.shape == (0,) and dz.shape == (0, 20)


def test_same_bits_and_other_stream(ops):
    for n, v in ((600, 90), (50, 4000), (3, 40_000)):
        x = _inputs(n, v, 6, BF16, True)
        a = _run(ops, x, 2.0, 0.5)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            b = _run(ops, x, 2.0, 0.5)
        assert all(torch.equal(u, w) for u, w in zip(a, b))


def test_graph_replay(ops):
    x = {k: t.to(DEV) for k, t in _inputs(4, 30_000, 16, BF16, True).items()}

    def both():
        loss, stats = ops.distillation_loss(x["z"], x["t"], x["c"], x["lse"], x["labels"], 2.0, 0.5)
        return loss, ops.distillation_loss_backward(x["g"], x["z"], x["t"], x["c"], x["labels"], stats, 2.0, 0.5)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for k in range(3):
        x["z"].mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, both())), k


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_module_gradient_and_differences(ops, tail, reduction):
    from piecewiselinearembeddings_optimized_amd import CudaDistillationLoss

    x = _inputs(12, 60, 7, tail=tail)
    m = CudaDistillationLoss(2.0, 0.7, reduction)
    up = torch.randn(3, 4, generator=torch.Generator().manual_seed(0)) if reduction == "none" else torch.tensor(1.7)

    def value(z, dev, double=False):
        put = lambda t, *s: None if t is None else t.reshape(3, 4, *s).to(dev)  # noqa: E731
        out = m(z, put(x["t"], 7), put(x["c"], 7), put(x["lse"]), put(x["labels"]))
        return ((out.double() if double else out) * up.to(dev)).sum()

    z = x["z"].reshape(3, 4, 60).clone().requires_grad_()
    want = torch.autograd.grad(value(z, "cpu"), z)[0]
    zd = z.detach().to(DEV).requires_grad_()
    got = torch.autograd.grad(value(zd, DEV), zd)[0]
    torch.testing.assert_close(got.cpu(), want, rtol=1e-4, atol=1e-5)
    step, h = torch.randn_like(zd), 1e-2
    with torch.no_grad():
        slope = float(value(zd + h * step, DEV, True) - value(zd - h * step, DEV, True)) / (2 * h)
    along = float((got.double() * step).sum())
    # (third derivatives of the loss are at most T^2 (1 / T)^3 and 1, over 12 rows)
    assert abs(slope - along) < 1e-2 * (1 + abs(along))


def test_opcheck(ops):
    x = {k: t.to(DEV) for k, t in _inputs(5, 30, 4, tail=True).items()}
    z = x["z"].requires_grad_()
    torch.library.opcheck(ops.distillation_loss.default, (z, x["t"], x["c"], x["lse"], x["labels"], 2.0, 0.5))
    torch.library.opcheck(ops.distillation_loss.default, (z, x["t"], x["c"], None, None, 1.0, 1.0))


def test_compiled(ops):
    from piecewiselinearembeddings_optimized_amd import CudaDistillationLoss

    x = {k: None if t is None else t.to(DEV) for k, t in _inputs(5, 30, 4).items()}
    m, z = CudaDistillationLoss(2.0, 0.5), x["z"].requires_grad_()
    f = lambda z: m(z * 2, x["t"], x["c"], labels=x["labels"])  # noqa: E731
    got = torch.autograd.grad(torch.compile(f, fullgraph=True)(z), z)[0]
    torch.testing.assert_close(got, torch.autograd.grad(f(z), z)[0])


def test_refusals(ops):
    x = {k: t.to(DEV) for k, t in _inputs(5, 30, 4, tail=True).items()}

    def call(z=x["z"], t=x["t"], c=x["c"], lse=x["lse"], labels=x["labels"], temperature=2.0, alpha=0.5):
        return ops.distillation_loss(z, t, c, lse, labels, temperature, alpha)

    for match, kw in {
        "shape \\[N, V\\]": {"z": x["z"][0]},
        "logits must be float32": {"z": x["z"].double()},
        "logits must be contiguous": {"z": torch.randn(30, 5, device=DEV).T},
        "teacher_logits must have shape": {"t": x["t"][:3]},
        "teacher_classes must have shape": {"c": x["c"][:, :2].contiguous()},
        "teacher_classes must be int32 or int64": {"c": x["c"].float()},
        "labels must be int64": {"labels": x["labels"].int()},
        "teacher_lse must be float32": {"lse": x["lse"].double()},
        "temperature must be between": {"temperature": 0.0},
        "alpha must be between": {"alpha": 1.5},
        "same CUDA device": {"t": x["t"].cpu()},
    }.items():
        with pytest.raises(RuntimeError, match=match):
            call(**kw)
    with pytest.raises(RuntimeError, match="temperature"):
        call(temperature=float("nan"))
    with pytest.raises(RuntimeError, match="grad_loss must be"):
        ops.distillation_loss_backward(x["g"].double(), x["z"], x["t"], x["c"], None, torch.zeros(5, 8, device=DEV), 1.0, 1.0)


def test_c_abi(ops):
    """The ctypes binding gives the operators' bits, and refuses a small workspace."""
    from piecewiselinearembeddings_optimized_amd import capi

    x = _inputs(3, 30_000, 9, BF16, True)
    want = _run(ops, x, 2.0, 0.5)
    dev = {k: t.to(DEV) for k, t in x.items()}
    loss, stats, dz = torch.empty(3, device=DEV), torch.empty(3, 8, device=DEV), torch.empty_like(dev["z"])
    kw = {"labels": dev["labels"], "temperature": 2.0, "alpha": 0.5}
    capi.distill(dev["z"], dev["t"], dev["c"], loss, stats, teacher_lse=dev["lse"], **kw)
    capi.distill_backward(dev["g"], dev["z"], dev["t"], dev["c"], stats, dz, **kw)
    assert torch.equal(loss.cpu(), want[0]) and torch.equal(dz.cpu(), want[1])
    with pytest.raises(capi.PleError, match="workspace"):
        capi.distill(dev["z"], dev["t"], dev["c"], loss, stats, workspace=torch.empty(16, dtype=torch.uint8, device=DEV))

"""What a model has around its numerical embeddings: embeddings of tokens and
categorical columns, the norms of a residual trunk, and the loss of a student
that learns from a larger teacher's top logits.

On a HIP device the modules run the operators ``lookup``, ``residual_norm`` and
``distillation_loss`` of ``torch.ops.rtdl_num_embeddings_cuda`` (sums over rows in
a fixed order); on the CPU the same formulas run as ordinary PyTorch operations.
Tensors are float32, float16 or bfloat16, computed in 32 bits; on the CPU float64
too, computed in 64 bits (a device refuses it).  First-order autograd and
``torch.compile(fullgraph=True)`` work; double backward is not implemented.
"""

from __future__ import annotations

from typing import Literal

import torch
from torch import Tensor, nn
from torch.nn.parameter import Parameter

from ._meta import NORM_MAX_WIDTH

_ops = torch.ops.rtdl_num_embeddings_cuda

_NORMS = {None: 0, "rms": 1, "layer": 2}
_ACTIVATIONS = {None: 0, "sigmoid": 1, "tanh": 2}


def _compute_dtype(t: Tensor) -> torch.dtype:
    """The autocast dtype of the device of ``t``, else the dtype of ``t``."""
    if torch.is_autocast_enabled(t.device.type):
        return torch.get_autocast_dtype(t.device.type)
    return t.dtype


def _wide(t: Tensor) -> Tensor:
    """``t`` in the type the CPU computes in."""
    return t if t.dtype == torch.float64 else t.float()


# ---------------------------------------------------------------------------
# lookup
# ---------------------------------------------------------------------------

def _lookup_cpu(tokens: Tensor, weight: Tensor, offsets: Tensor | None, scale: float, padding_idx: int,
                dtype: torch.dtype) -> Tensor:
    tokens = tokens.long()
    sizes = weight.shape[0] if offsets is None else offsets.diff()
    row = tokens if offsets is None else tokens + offsets[:-1]
    missing, beyond = tokens < 0, tokens >= sizes
    out = _wide(weight[torch.where(missing | beyond, 0, row)]) * scale
    if padding_idx >= 0:
        out = torch.where((tokens == padding_idx)[..., None], out.detach(), out)
    out = torch.where(missing[..., None], 0.0, torch.where(beyond[..., None], float("nan"), out))
    return out.to(dtype)


def _lookup(tokens, weight, offsets, scale, padding_idx) -> Tensor:
    dtype = _compute_dtype(weight)
    if weight.device.type != "cuda":
        return _lookup_cpu(tokens, weight, offsets, scale, padding_idx, dtype)
    return _ops.lookup(tokens.contiguous(), weight, offsets, scale, padding_idx, dtype)


class CudaTokenEmbeddings(nn.Module):
    """Scaled rows of a table: ``scale * weight[token]`` for tokens of any shape.

    ``scale`` is applied in 32 bits before the one rounding to the output's
    dtype (the weight's, or the autocast dtype).  A negative token is missing:
    a row of zeros without a gradient.  A token beyond the table gives a row of
    NaN.  ``padding_idx``: a token whose row gets no gradient.
    """

    def __init__(self, n_tokens: int, d_embedding: int, *, scale: float = 1.0, padding_idx: int | None = None) -> None:
        if n_tokens <= 0 or d_embedding <= 0:
            raise ValueError(f"n_tokens and d_embedding must be positive, got {n_tokens} and {d_embedding}")
        if padding_idx is not None and not 0 <= padding_idx < n_tokens:
            raise ValueError(f"padding_idx must be in [0, {n_tokens}), got {padding_idx}")
        super().__init__()
        self.scale = float(scale)
        self.padding_idx = padding_idx
        self.weight = Parameter(torch.empty(n_tokens, d_embedding))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        nn.init.normal_(self.weight, std=self.weight.shape[1] ** -0.5)

    def forward(self, tokens: Tensor) -> Tensor:
        return _lookup(tokens, self.weight, None, self.scale, -1 if self.padding_idx is None else self.padding_idx)


class CudaCategoricalEmbeddings(nn.Module):
    """Embeddings of categorical columns ``[..., F] -> [..., F, d]``, next to
    the numerical ones.

    Column ``f`` has categories ``0 .. cardinalities[f] - 1``; the columns'
    tables are the rows of one ``weight``.  A negative category is a missing
    value: a row of zeros without a gradient.  A category beyond its column's
    gives a row of NaN.
    """

    def __init__(self, cardinalities: list[int], d_embedding: int, *, scale: float = 1.0) -> None:
        if not cardinalities or min(cardinalities) <= 0 or d_embedding <= 0:
            raise ValueError("cardinalities (at least one) and d_embedding must be positive, "
                             f"got {cardinalities} and {d_embedding}")
        super().__init__()
        self.scale = float(scale)
        self.weight = Parameter(torch.empty(sum(cardinalities), d_embedding))
        self.register_buffer("offsets", torch.tensor([0, *cardinalities]).cumsum(0), persistent=False)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        bound = self.weight.shape[1] ** -0.5
        nn.init.uniform_(self.weight, -bound, bound)

    def get_output_shape(self) -> torch.Size:
        return torch.Size((self.offsets.shape[0] - 1, self.weight.shape[1]))

    def forward(self, tokens: Tensor) -> Tensor:
        if tokens.shape[-1:] != (self.offsets.shape[0] - 1,):
            raise ValueError(f"Expected {self.offsets.shape[0] - 1} categorical features, got shape {tuple(tokens.shape)}")
        return _lookup(tokens, self.weight, self.offsets, self.scale, -1)


# ---------------------------------------------------------------------------
# residual norm
# ---------------------------------------------------------------------------

def _norm_cpu(x: Tensor, kind: str, weight: Tensor | None, bias: Tensor | None, eps: float) -> Tensor:
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        x = x * _wide(weight)
    return x if bias is None else x + _wide(bias)


class CudaResidualNorm(nn.Module):
    """The norms after and before a block of a residual trunk, with the block's
    gate and the residual scale, in one pass over the rows:

        stream = residual_scale * residual + h(gate) * post_norm(branch)
        normed = pre_norm(stream)

    ``forward(residual, branch)`` returns ``(stream, normed)``: the trunk's new
    residual and the next block's input.  Without a branch (the trunk's start)
    it returns ``(residual, pre_norm(residual))``.  Norms: ``None``, ``"rms"`` or
    ``"layer"``, with learned weights (and biases with ``bias=True``); with
    ``pre_norm=None`` (the trunk's end) ``normed`` is the stream itself.

    ``gate``: ``None``, or ``"learned"`` for one learned value a channel
    (``gate_init``); a gate made by the model is passed to ``forward`` with the
    residual's trailing width and any leading shape that broadcasts over the
    rows in groups: ``[D]``, ``[B, 1, D]`` or the residual's own.  ``gate_activation``:
    ``None``, ``"sigmoid"`` or ``"tanh"``.

    The stream keeps the residual's dtype (float32 for a trunk under autocast),
    ``normed`` has the branch's; means and factors are 32-bit.
    """

    def __init__(self, d: int, *, post_norm: Literal[None, "rms", "layer"] = None,
                 pre_norm: Literal[None, "rms", "layer"] = "rms", bias: bool = False,
                 gate: Literal[None, "learned"] = None, gate_init: float = 1.0,
                 gate_activation: Literal[None, "sigmoid", "tanh"] = None, residual_scale: float = 1.0,
                 eps: float = 1e-5) -> None:
        if not 0 < d <= NORM_MAX_WIDTH:
            raise ValueError(f"d must be between 1 and {NORM_MAX_WIDTH}, got {d}")
        if post_norm not in _NORMS or pre_norm not in _NORMS:
            raise ValueError(f'norms must be None, "rms" or "layer", got {post_norm!r} and {pre_norm!r}')
        if gate_activation not in _ACTIVATIONS:
            raise ValueError(f'gate_activation must be None, "sigmoid" or "tanh", got {gate_activation!r}')
        if gate not in (None, "learned"):
            raise ValueError(f'gate must be None or "learned", got {gate!r}')
        super().__init__()
        self.d, self.post_norm, self.pre_norm = d, post_norm, pre_norm
        self.gate_activation, self.residual_scale, self.eps = gate_activation, float(residual_scale), float(eps)
        for name, kind in (("post", post_norm), ("pre", pre_norm)):
            self.register_parameter(f"{name}_weight", None if kind is None else Parameter(torch.ones(d)))
            self.register_parameter(f"{name}_bias", Parameter(torch.zeros(d)) if kind is not None and bias else None)
        self.register_parameter("gate", None if gate is None else Parameter(torch.full((1, d), float(gate_init))))

    def _gate_rows(self, gate: Tensor | None, residual: Tensor) -> Tensor | None:
        """The gate as [G, D], each row for an equal share of consecutive rows."""
        if gate is None:
            return self.gate
        if self.gate is not None:
            raise ValueError("this module has a learned gate; forward takes no other")
        if gate.shape[-1:] != (self.d,) or gate.ndim > residual.ndim:
            raise ValueError(f"gate of shape {tuple(gate.shape)} does not fit rows of shape {tuple(residual.shape)}")
        lead = (1,) * (residual.ndim - gate.ndim) + tuple(gate.shape[:-1])
        shared = False
        for g, n in zip(lead, residual.shape[:-1]):
            if g == n and not shared:
                continue
            if g != 1:
                raise ValueError(f"gate of shape {tuple(gate.shape)} does not broadcast over rows of shape "
                                 f"{tuple(residual.shape)} in groups of consecutive rows")
            shared = True
        weight = self.post_weight if self.pre_weight is None else self.pre_weight
        # (under autocast a gate has the autocast dtype, the weights theirs)
        return (gate if weight is None else gate.to(weight.dtype)).reshape(-1, self.d).contiguous()

    def forward(self, residual: Tensor, branch: Tensor | None = None, gate: Tensor | None = None) -> tuple[Tensor, Tensor]:
        if residual.shape[-1:] != (self.d,):
            raise ValueError(f"Expected rows of {self.d} elements, got shape {tuple(residual.shape)}")
        if branch is None:
            if gate is not None:
                raise ValueError("a gate needs a branch")
            if self.pre_norm is None:
                return residual, residual
            return residual, self._run(residual, None, None, None, 1.0, _compute_dtype(residual))[1]
        stream, normed = self._run(residual, branch, self._gate_rows(gate, residual), self.post_norm, self.residual_scale,
                                   branch.dtype)
        return stream, stream if self.pre_norm is None else normed

    def _run(self, residual, branch, gate, post_norm, residual_scale, dtype):
        after = post_norm is not None
        post = (self.post_weight, self.post_bias) if after else (None, None)
        if residual.device.type != "cuda":
            stream = residual
            if branch is not None:
                p = _wide(branch)
                if after:
                    p = _norm_cpu(p, post_norm, *post, self.eps)
                if gate is not None:
                    h = {None: lambda t: t, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[self.gate_activation](_wide(gate))
                    groups = max(1, gate.shape[0])
                    p = (p.reshape(groups, -1, self.d) * h[:, None]).reshape(p.shape)
                stream = (residual_scale * _wide(residual) + p).to(residual.dtype)
            if self.pre_norm is None:
                return stream, None
            return stream, _norm_cpu(_wide(stream), self.pre_norm, self.pre_weight, self.pre_bias, self.eps).to(dtype)
        stream, normed, _ = _ops.residual_norm(
            residual.contiguous(), None if branch is None else branch.contiguous(), *post, gate, self.pre_weight,
            self.pre_bias, _NORMS[post_norm], _NORMS[self.pre_norm], _ACTIVATIONS[self.gate_activation], residual_scale,
            self.eps, dtype)
        return stream, normed


# ---------------------------------------------------------------------------
# distillation loss
# ---------------------------------------------------------------------------

def _distill_cpu(logits, teacher_logits, classes, teacher_lse, labels, temperature, alpha) -> Tensor:
    z = _wide(logits)
    n, v = z.shape
    live = ~torch.isneginf(z).all(-1)
    z = torch.where(live[:, None], z, 0.0)
    classes = classes.long()
    known = (classes >= 0) & (classes < v)
    c = torch.where(known, classes, 0)
    log_q = torch.log_softmax(z / temperature, -1)
    t = torch.where(classes >= 0, teacher_logits.detach().to(z.dtype) / temperature, -torch.inf)
    taught = (classes >= 0).any(-1)
    if teacher_lse is None:
        taught = taught & ~torch.isneginf(t).all(-1)
        lse = torch.where(taught, torch.logsumexp(torch.where(taught[:, None], t, 0.0), -1), 0.0)
    else:
        lse = teacher_lse.detach().to(z.dtype)
    log_p = t - lse[:, None]
    p = log_p.exp()
    q_at = log_q.gather(1, c)
    kd = torch.where(known & (p > 0), p * (torch.where(p > 0, log_p, 0.0) - torch.where(p > 0, q_at, 0.0)), 0.0).sum(-1)
    if teacher_lse is not None:
        inside = torch.zeros(n, v, dtype=torch.int32)
        inside.scatter_add_(1, c, known.int())
        # (in logarithms: a student's outside mass may be below what 32 bits hold; a row
        # whose other classes are all masked has none, and the log-sum of nothing has a
        # gradient of NaN)
        outside = log_q.masked_fill(inside != 0, -torch.inf)
        none = torch.isneginf(outside).all(-1)
        log_outside = torch.where(none, -torch.inf, torch.logsumexp(torch.where(none[:, None], 0.0, outside), -1))
        rho = (1 - p.sum(-1)).clamp_min(0)
        some = taught & (rho > 0) & (log_outside > -700)
        kd = kd + torch.where(some, rho * (torch.where(some, rho, 1.0).log() - torch.where(some, log_outside, 0.0)), 0.0)
    kd = torch.where(taught, kd, 0.0)
    # (a product: the gradient is NaN too)
    kd = kd * torch.where((classes >= v).any(-1), torch.nan, 1.0)
    loss = alpha * temperature ** 2 * kd if alpha > 0 else z.new_zeros(n)
    if labels is not None and alpha < 1:
        ce = -torch.log_softmax(z, -1).gather(1, labels.clamp(0, v - 1)[:, None])[:, 0]
        loss = loss + (1 - alpha) * torch.where(labels >= 0, ce, 0.0) * torch.where(labels >= v, torch.nan, 1.0)
    return torch.where(live, loss, 0.0)


class CudaDistillationLoss(nn.Module):
    """Loss of a student against a larger teacher's top logits, and hard labels.

    ``forward(logits, teacher_logits, teacher_classes, teacher_lse=None,
    labels=None)``: the student's logits ``[..., V]``, the teacher's ``K`` top
    logits ``[..., K]`` and their classes.  With ``q = softmax(logits / T)`` and
    ``p = exp(teacher_logits / T - l)`` a row's loss is

        alpha * T^2 * KL(p || q) + (1 - alpha) * cross_entropy(logits, label)

    ``l`` normalises the K logits, or is ``teacher_lse``, the log-sum of the
    exponentials of ``t / T`` over the teacher's whole vocabulary: then the mass
    that the K classes leave out is one more outcome, for the teacher and for
    the student.  Negative classes and labels are absent; without ``labels`` the
    loss is the first term.  ``reduction``: ``"mean"`` (over the rows), ``"sum"``
    or ``"none"``.  The teacher gets no gradient.
    """

    def __init__(self, temperature: float = 1.0, alpha: float = 1.0,
                 reduction: Literal["mean", "sum", "none"] = "mean") -> None:
        if not 1e-6 < temperature < 1e6:
            raise ValueError(f"temperature must be between 1e-6 and 1e6, got {temperature}")
        if not 0.0 <= alpha <= 1.0:
            raise ValueError(f"alpha must be between 0 and 1, got {alpha}")
        if reduction not in ("mean", "sum", "none"):
            raise ValueError(f'reduction must be "mean", "sum" or "none", got {reduction!r}')
        super().__init__()
        self.temperature, self.alpha, self.reduction = float(temperature), float(alpha), reduction

    def forward(self, logits: Tensor, teacher_logits: Tensor, teacher_classes: Tensor, teacher_lse: Tensor | None = None,
                labels: Tensor | None = None) -> Tensor:
        if logits.ndim < 1 or teacher_logits.shape[:-1] != logits.shape[:-1]:
            raise ValueError(f"teacher_logits of shape {tuple(teacher_logits.shape)} do not fit logits of shape "
                             f"{tuple(logits.shape)}")
        lead = logits.shape[:-1]
        args = (logits.reshape(-1, logits.shape[-1]), teacher_logits.reshape(-1, teacher_logits.shape[-1]),
                teacher_classes.reshape(-1, teacher_classes.shape[-1]),
                None if teacher_lse is None else teacher_lse.reshape(-1),
                None if labels is None else labels.reshape(-1))
        if logits.device.type != "cuda":
            loss = _distill_cpu(*args, self.temperature, self.alpha)
        else:
            loss, _ = _ops.distillation_loss(*(None if t is None else t.contiguous() for t in args), self.temperature,
                                             self.alpha)
        if self.reduction == "none":
            return loss.reshape(lead)
        return loss.mean() if self.reduction == "mean" else loss.sum()

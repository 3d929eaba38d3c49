"""What the blocks of a model on embedded columns or tokens need next to its
linear layers: the norm of groups of channels with its activation, and the
learned bias of attention scores by relative position.

On a HIP device the modules run the operators ``group_norm`` and
``relative_bias`` of ``torch.ops.rtdl_num_embeddings_cuda`` (sums in a fixed
order); on the CPU the same formulas run as ordinary PyTorch operations.  Tensors
are float32, float16 or bfloat16, computed in 32 bits; on the CPU float64 too,
computed in 64 bits (a device refuses it).  First-order autograd and
``torch.compile(fullgraph=True)`` work; double backward is not implemented.
"""

from __future__ import annotations

from typing import Literal

import torch
from torch import Tensor, nn
from torch.nn.parameter import Parameter

from .trunk import _compute_dtype, _wide

_ops = torch.ops.rtdl_num_embeddings_cuda

_ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


# ---------------------------------------------------------------------------
# group norm
# ---------------------------------------------------------------------------

def _group_norm_cpu(x: Tensor, weight: Tensor | None, bias: Tensor | None, groups: int, activation: str | None,
                    eps: float) -> Tensor:
    z = _wide(x)
    if x.numel() > 0:
        z = z.reshape(x.shape[0], -1, groups, x.shape[-1] // groups)
        z = z - z.mean((1, 3), keepdim=True)
        z = (z * torch.rsqrt(z.square().mean((1, 3), keepdim=True) + eps)).reshape(x.shape)
    if weight is not None:
        z = z * _wide(weight)
    if bias is not None:
        z = z + _wide(bias)
    if activation == "relu":
        z = torch.relu(z)
    elif activation == "silu":
        z = z * torch.sigmoid(z)
    elif activation == "gelu":
        z = 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    return z.to(x.dtype)


class CudaGroupNorm(nn.Module):
    """Group norm and an activation of rows whose channels are last in memory,
    ``[N, ..., C] -> [N, ..., C]``, in one pass where a sample's groups fit a
    workgroup's registers:

        y = activation((x - mean) / sqrt(var + eps) * weight + bias)

    The ``C`` channels are ``num_groups`` groups of adjacent ones; mean and
    variance (biased) are a sample's over all of its positions and the group's
    channels.  ``[N, F, d]`` embeddings are such rows, and so is
    ``x.movedim(1, -1)`` of a ``torch.channels_last`` tensor ``[N, C, H, W]``.
    ``activation``: ``None``, ``"relu"``, ``"silu"`` or ``"gelu"`` (by the error
    function).  The output has the input's dtype; statistics are 32-bit.
    """

    def __init__(self, num_groups: int, num_channels: int, *, activation: Literal[None, "relu", "silu", "gelu"] = None,
                 affine: bool = True, eps: float = 1e-5) -> None:
        if num_groups <= 0 or num_channels <= 0 or num_channels % num_groups:
            raise ValueError(f"num_groups must divide num_channels, got {num_groups} and {num_channels}")
        if activation not in _ACTIVATIONS:
            raise ValueError(f'activation must be None, "relu", "silu" or "gelu", got {activation!r}')
        super().__init__()
        self.num_groups, self.num_channels, self.activation, self.eps = num_groups, num_channels, activation, float(eps)
        self.register_parameter("weight", Parameter(torch.ones(num_channels)) if affine else None)
        self.register_parameter("bias", Parameter(torch.zeros(num_channels)) if affine else None)

    def forward(self, x: Tensor) -> Tensor:
        if x.ndim < 2 or x.shape[-1] != self.num_channels:
            raise ValueError(f"Expected [N, ..., {self.num_channels}], got shape {tuple(x.shape)}")
        if x.device.type != "cuda":
            return _group_norm_cpu(x, self.weight, self.bias, self.num_groups, self.activation, self.eps)
        return _ops.group_norm(x.contiguous(), self.weight, self.bias, self.num_groups, _ACTIVATIONS[self.activation],
                               self.eps)[0]


# ---------------------------------------------------------------------------
# relative position bias
# ---------------------------------------------------------------------------

def relative_buckets(num_buckets: int, max_distance: int, bidirectional: bool = True) -> Tensor:
    """The bucket of every distance ``key - query`` from ``-max_distance`` to
    ``max_distance`` (what is further counts as that far), int32.

    ``bidirectional``: the first half of the buckets for keys at or before the
    query, the second for keys after it; else all of them for the past, and
    bucket 0 for the future.  Half of a side's ``n`` buckets hold one distance
    each, the others begin at the first whole number that is at least
    ``e * (max_distance / e) ** (j / (n - e))``, ``e = n // 2`` -- in whole
    numbers, so that no logarithm's rounding moves a border.
    """
    side = num_buckets // 2 if bidirectional else num_buckets
    if side < 1:
        raise ValueError(f"there has to be a bucket for each side, got {num_buckets}")
    exact = side // 2
    steps = side - exact
    if max_distance < max(1, exact + (steps > 1)):
        raise ValueError(f"max_distance must exceed the {exact} distances with buckets of their own, got {max_distance}")
    borders = list(range(exact + 1))
    for j in range(1, steps if exact else 1):
        # the least d with d ** steps >= exact ** (steps - j) * max_distance ** j
        power = exact ** (steps - j) * max_distance ** j
        d = max(1, int(exact * (max_distance / exact) ** (j / steps)) - 1)
        while d ** steps < power:
            d += 1
        while (d - 1) ** steps >= power:
            d -= 1
        borders.append(d)
    past = torch.bucketize(torch.arange(max_distance + 1), torch.tensor(borders), right=True) - 1
    future = past[1:] + side if bidirectional else torch.zeros(max_distance, dtype=torch.long)
    return torch.cat([past.flip(0), future]).to(torch.int32)


def _relative_bias_cpu(weight: Tensor, buckets: Tensor, starts: Tensor | None, q_len: int, k_len: int, offset: int,
                       causal: bool, dtype: torch.dtype) -> Tensor:
    far = buckets.shape[0] // 2
    first = torch.tensor([offset]) if starts is None else starts.long().clamp(-2 ** 60, 2 ** 60)    # (so that no difference overflows)
    d = torch.arange(k_len) - (first[:, None, None] + torch.arange(q_len)[:, None])          # [B, q, k]
    row = buckets[d.clamp(-far, far) + far].long()
    none, beyond = row < 0, row >= weight.shape[0]
    out = _wide(weight)[torch.where(none | beyond, 0, row)]
    out = torch.where(none[..., None], 0.0, out)
    out = torch.where(beyond[..., None], torch.nan, out).movedim(-1, 1)
    if causal:
        out = torch.where((d > 0)[:, None], -torch.inf, out)
    out = out.to(dtype).contiguous()
    return out[0] if starts is None else out


class CudaRelativeBias(nn.Module):
    """A learned bias of attention scores by the distance of key and query.

    ``forward(q_len, k_len)`` gives ``[H, q_len, k_len]``, to be added to scores
    (or passed as an attention mask): row ``buckets[key - query]`` of the learned
    ``weight [num_buckets, H]``.  The queries are the last of the keys
    (``offset = k_len - q_len``) unless ``offset`` says where the first one
    stands.  ``starts`` (int64 ``[B]``) gives it for every sample, for sequences of
    different lengths: the result is ``[B, H, q_len, k_len]``.

    The buckets are :func:`relative_buckets`' (``max_distance``,
    ``bidirectional``), or ``buckets``: int32 ``[2 * far + 1]``, the row of each
    distance from ``-far`` to ``far``; a negative one has no bias, one beyond the
    table gives NaN.  ``causal``: keys after the query have ``-inf``.

    The output has the weight's dtype, the autocast dtype, or ``dtype``.
    """

    def __init__(self, num_buckets: int, num_heads: int, *, max_distance: int = 128, bidirectional: bool = True,
                 causal: bool = False, buckets: Tensor | None = None) -> None:
        if num_buckets <= 0 or num_heads <= 0:
            raise ValueError(f"num_buckets and num_heads must be positive, got {num_buckets} and {num_heads}")
        if buckets is None:
            buckets = relative_buckets(num_buckets, max_distance, bidirectional)
        elif buckets.ndim != 1 or buckets.shape[0] < 3 or buckets.shape[0] % 2 == 0:
            raise ValueError(f"buckets must have shape [2 * far + 1], far at least 1, got {tuple(buckets.shape)}")
        super().__init__()
        self.causal = causal
        self.weight = Parameter(torch.empty(num_buckets, num_heads))
        self.register_buffer("buckets", buckets.to(torch.int32).contiguous(), persistent=False)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        nn.init.normal_(self.weight, std=self.weight.shape[1] ** -0.5)

    def forward(self, q_len: int, k_len: int | None = None, *, offset: int | None = None, starts: Tensor | None = None,
                dtype: torch.dtype | None = None) -> Tensor:
        k_len = q_len if k_len is None else k_len
        if q_len < 0 or k_len < 0:
            raise ValueError(f"lengths must not be negative, got {q_len} and {k_len}")
        if starts is not None and (offset is not None or starts.ndim != 1):
            raise ValueError("starts must have shape [B], and takes the place of offset")
        dtype = _compute_dtype(self.weight) if dtype is None else dtype
        args = (starts, q_len, k_len, k_len - q_len if offset is None else offset, self.causal, dtype)
        if self.weight.device.type != "cuda":
            return _relative_bias_cpu(self.weight, self.buckets, *args)
        return _ops.relative_bias(self.weight, self.buckets, None if starts is None else starts.contiguous(), *args[1:])

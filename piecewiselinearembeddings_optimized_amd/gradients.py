"""The norm of a model's gradients together, and their clipping to a limit.

On a HIP device they run the operators ``gradient_norm``, ``clip_gradients_`` and
``clip_gradients_into`` of ``torch.ops.rtdl_num_embeddings_cuda``: all tensors in a
few launches, sums in 64 bits and a fixed order, no synchronisation with the
host.  On the CPU the same formulas run as ordinary PyTorch operations.
"""

from __future__ import annotations

from collections.abc import Iterable, Sequence

import torch
from torch import Tensor

_ops = torch.ops.rtdl_num_embeddings_cuda


def _norm_cpu(grads: Sequence[Tensor], norm_type: float) -> Tensor:
    wide = [g.double() for g in grads if g.numel() > 0]
    if not wide:
        total = torch.zeros((), dtype=torch.float64)
    elif norm_type == 2.0:
        total = torch.stack([g.square().sum() for g in wide]).sum().sqrt()
    elif norm_type == 1.0:
        total = torch.stack([g.abs().sum() for g in wide]).sum()
    else:
        total = torch.stack([g.abs().max() for g in wide]).max()
    return total.float()


def _check(grads: Sequence[Tensor], norm_type: float, max_norm: float = 0.0) -> None:
    if norm_type not in (1.0, 2.0, float("inf")):
        raise ValueError(f"norm_type must be 1, 2 or infinity, got {norm_type}")
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    for g in grads:
        if g.is_sparse or g.is_complex():
            raise ValueError("gradients must be dense and real")


@torch.no_grad()
def gradient_norm(grads: Sequence[Tensor], norm_type: float = 2.0) -> Tensor:
    """The norm of all elements of all tensors together, a float32 scalar tensor:
    ``norm_type`` 1, 2 or infinity (the largest absolute value); NaN if an element
    is.  0 without tensors."""
    grads = list(grads)
    norm_type = float(norm_type)
    if not grads:
        return torch.zeros(())
    if grads[0].device.type == "cuda":
        return _ops.gradient_norm(grads, norm_type)
    _check(grads, norm_type)
    return _norm_cpu(grads, norm_type)


@torch.no_grad()
def clip_gradients_(grads: Sequence[Tensor], max_norm: float, norm_type: float = 2.0, *, norm: Tensor | None = None,
                    out: Sequence[Tensor] | None = None) -> Tensor:
    """Multiplies all tensors by ``min(1, max_norm / (norm + 1e-6))`` and returns
    their norm (:func:`gradient_norm`).

    In place, where nothing is written if the factor is 1; or into ``out``, a tensor
    of the same shape and layout and any of the three dtypes for each (an
    optimizer's 32-bit gradients from a model's 16-bit ones).  Tensors that are
    written must not share memory.  ``norm``: a norm that is known already, as a
    float32 tensor -- the norm over all ranks of sharded gradients, say.  An
    infinite ``max_norm`` clips nothing; with a norm of infinity the factor is 0,
    with NaN it is NaN.
    """
    grads = list(grads)
    max_norm, norm_type = float(max_norm), float(norm_type)
    if not grads:
        return torch.zeros(()) if norm is None else norm.clone()
    if grads[0].device.type == "cuda":
        if out is None:
            return _ops.clip_gradients_(grads, max_norm, norm_type, norm)
        return _ops.clip_gradients_into(grads, list(out), max_norm, norm_type, norm)
    _check(grads, norm_type, max_norm)
    out = grads if out is None else list(out)
    if len(out) != len(grads):
        raise ValueError("out must have a tensor for every gradient")
    if any(o.shape != g.shape for g, o in zip(grads, out)):
        raise ValueError("out must have the shape of its gradient")
    # (of those that overlap in part, a device finds all; in a graph tensors have no addresses yet)
    begins = [] if torch.compiler.is_compiling() else [o.data_ptr() for o in out if o.numel() > 0 and not o.is_meta]
    if len(set(begins)) < len(begins):
        raise ValueError("gradients that are scaled must not share memory with each other or with out")
    norm = _norm_cpu(grads, norm_type) if norm is None else norm.reshape(()).clone()
    factor = torch.ones(()) if max_norm == float("inf") else (max_norm / (norm.double() + 1e-6)).clamp_max(1.0).float()
    for g, o in zip(grads, out):
        if o is not g or factor != 1:
            wide = g if g.dtype == torch.float64 else g.float()
            o.copy_(wide * factor)
    return norm


def clip_grad_norm_(parameters: Tensor | Iterable[Tensor], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: bool | None = None) -> Tensor:
    """:func:`clip_gradients_` of the parameters' gradients, with the arguments of
    ``torch.nn.utils.clip_grad_norm_`` (``norm_type`` 1, 2 or infinity).  A parameter
    that is given twice counts once.  ``error_if_nonfinite`` waits for the norm and
    raises where it is not finite, before anything is scaled.  ``foreach`` changes
    nothing: a device takes all gradients together in any case."""
    parameters = [parameters] if isinstance(parameters, Tensor) else list(parameters)
    grads = list({id(p): p.grad for p in parameters if p.grad is not None}.values())
    norm = None
    if error_if_nonfinite:
        norm = gradient_norm(grads, norm_type)
        if not bool(torch.isfinite(norm)):
            raise RuntimeError(f"the gradients' norm of order {norm_type} is not finite; nothing was clipped")
    return clip_gradients_(grads, max_norm, norm_type, norm=norm)

"""FakeTensor (meta) kernels of the PLE operators.

They state the shape / dtype contract of every operator without touching
data, so ``torch.compile(fullgraph=True)`` and meta-device tracing work.  The
checks and messages of ``forward`` / ``backward`` follow the reference
(``src/rtdl_num_embeddings_cuda/_meta.py:22-188``); the ``*_with_bias`` and
``*_epilogue`` operators are this build's fused variants.
"""

from __future__ import annotations

import torch
from torch import Tensor

SUPPORTED_OUTPUT_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


def bin_indices_dtype(max_n_bins: int) -> torch.dtype:
    """uint8 up to 256 bins, int16 up to 32768, int32 beyond (``_meta.py:14-19``)."""
    if max_n_bins <= 256:
        return torch.uint8
    if max_n_bins <= 32768:
        return torch.int16
    return torch.int32


def _check_forward_inputs(x, bin_edges, inv_bin_widths, n_bins, weight) -> None:
    torch._check(x.ndim == 2, lambda: "x must have shape [N, F]")
    torch._check(bin_edges.ndim == 2, lambda: "bin_edges must have shape [F, B + 1]")
    torch._check(inv_bin_widths.ndim == 2, lambda: "inv_bin_widths must have shape [F, B]")
    torch._check(n_bins.ndim == 1, lambda: "n_bins must have shape [F]")
    torch._check(weight.ndim == 3, lambda: "weight must have shape [F, B, D]")
    f_count, max_n_bins = weight.shape[0], weight.shape[1]
    torch._check(x.shape[1] == f_count, lambda: "x.shape[1] must equal weight.shape[0]")
    torch._check(bin_edges.shape[0] == f_count, lambda: "bin_edges.shape[0] must equal weight.shape[0]")
    torch._check(bin_edges.shape[1] == max_n_bins + 1, lambda: "bin_edges.shape[1] must equal weight.shape[1] + 1")
    torch._check(inv_bin_widths.shape[0] == f_count, lambda: "inv_bin_widths.shape[0] must equal weight.shape[0]")
    torch._check(inv_bin_widths.shape[1] == max_n_bins, lambda: "inv_bin_widths.shape[1] must equal weight.shape[1]")
    torch._check(n_bins.shape[0] == f_count, lambda: "n_bins.shape[0] must equal weight.shape[0]")
    torch._check(x.dtype == torch.float32, lambda: "x must be float32")
    torch._check(bin_edges.dtype == torch.float32, lambda: "bin_edges must be float32")
    torch._check(inv_bin_widths.dtype == torch.float32, lambda: "inv_bin_widths must be float32")
    torch._check(n_bins.dtype == torch.int32, lambda: "n_bins must be int32")
    torch._check(weight.dtype == torch.float32, lambda: "weight must be float32")


def _forward_outputs(x: Tensor, weight: Tensor, output_dtype: torch.dtype) -> tuple[Tensor, Tensor]:
    out = torch.empty((x.shape[0], x.shape[1], weight.shape[2]), dtype=output_dtype, device=x.device)
    idx = torch.empty((x.shape[0], x.shape[1]), dtype=bin_indices_dtype(weight.shape[1]), device=x.device)
    return out, idx


@torch.library.register_fake("rtdl_num_embeddings_cuda::forward")
def _forward_fake(x, bin_edges, inv_bin_widths, n_bins, weight, output_dtype):
    _check_forward_inputs(x, bin_edges, inv_bin_widths, n_bins, weight)
    torch._check(output_dtype in SUPPORTED_OUTPUT_DTYPES, lambda: "Unsupported output dtype")
    return _forward_outputs(x, weight, output_dtype)


@torch.library.register_fake("rtdl_num_embeddings_cuda::forward_with_bias")
def _forward_with_bias_fake(x, bin_edges, inv_bin_widths, n_bins, weight, bias, quant_dtype):
    _check_forward_inputs(x, bin_edges, inv_bin_widths, n_bins, weight)
    torch._check(quant_dtype in SUPPORTED_OUTPUT_DTYPES, lambda: "Unsupported quant dtype")
    torch._check(bias.ndim == 2, lambda: "bias must have shape [F, D]")
    torch._check(bias.shape[0] == weight.shape[0], lambda: "bias must have shape [F, D]")
    torch._check(bias.shape[1] == weight.shape[2], lambda: "bias must have shape [F, D]")
    torch._check(bias.dtype == torch.float32, lambda: "bias must be float32")
    return _forward_outputs(x, weight, torch.float32)


def _check_backward_inputs(grad_output, x, weight, bin_indices) -> None:
    torch._check(grad_output.ndim == 3, lambda: "grad_output must have shape [N, F, D]")
    torch._check(grad_output.shape[0] == x.shape[0], lambda: "grad_output N mismatch")
    torch._check(grad_output.shape[1] == x.shape[1], lambda: "grad_output F mismatch")
    torch._check(grad_output.shape[2] == weight.shape[2], lambda: "grad_output D mismatch")
    torch._check(bin_indices.shape[0] == x.shape[0], lambda: "bin_indices N mismatch")
    torch._check(bin_indices.shape[1] == x.shape[1], lambda: "bin_indices F mismatch")
    torch._check(bin_indices.dtype == bin_indices_dtype(weight.shape[1]), lambda: "bin_indices has an invalid dtype")
    torch._check(grad_output.dtype in SUPPORTED_OUTPUT_DTYPES, lambda: "Unsupported grad_output dtype")


def _maybe(t: Tensor, like: Tensor, wanted: bool) -> Tensor:
    return torch.empty_like(like) if wanted else torch.empty((0,), dtype=like.dtype, device=like.device)


@torch.library.register_fake("rtdl_num_embeddings_cuda::backward")
def _backward_fake(grad_output, x, bin_edges, inv_bin_widths, n_bins, weight, bin_indices,
                   compute_grad_x, compute_grad_weight):
    _check_backward_inputs(grad_output, x, weight, bin_indices)
    return _maybe(x, x, compute_grad_x), _maybe(weight, weight, compute_grad_weight)


@torch.library.register_fake("rtdl_num_embeddings_cuda::backward_with_bias")
def _backward_with_bias_fake(grad_output, x, bin_edges, inv_bin_widths, n_bins, weight, bin_indices,
                             quant_dtype, compute_grad_x, compute_grad_weight, compute_grad_bias):
    _check_backward_inputs(grad_output, x, weight, bin_indices)
    torch._check(quant_dtype in SUPPORTED_OUTPUT_DTYPES, lambda: "Unsupported quant dtype")
    grad_bias = (
        torch.empty((weight.shape[0], weight.shape[2]), dtype=weight.dtype, device=weight.device)
        if compute_grad_bias
        else torch.empty((0,), dtype=weight.dtype, device=weight.device)
    )
    return _maybe(x, x, compute_grad_x), _maybe(weight, weight, compute_grad_weight), grad_bias


def _check_fd(t, weight, name: str) -> None:
    torch._check(t.ndim == 2, lambda: f"{name} must have shape [F, D]")
    torch._check(t.shape[0] == weight.shape[0], lambda: f"{name} must have shape [F, D]")
    torch._check(t.shape[1] == weight.shape[2], lambda: f"{name} must have shape [F, D]")
    torch._check(t.dtype == torch.float32, lambda: f"{name} must be float32")


def _mask_words(d_embedding) -> int:
    return (d_embedding + 31) // 32


@torch.library.register_fake("rtdl_num_embeddings_cuda::forward_epilogue")
def _forward_epilogue_fake(x, bin_edges, inv_bin_widths, n_bins, weight, bias, lin_weight, lin_bias, relu,
                           save_mask, quant_dtype):
    _check_forward_inputs(x, bin_edges, inv_bin_widths, n_bins, weight)
    torch._check(quant_dtype in SUPPORTED_OUTPUT_DTYPES, lambda: "Unsupported quant dtype")
    torch._check((bias is None) != (lin_weight is None), lambda: "exactly one of bias and lin_weight must be given")
    if bias is not None:
        _check_fd(bias, weight, "bias")
    if lin_weight is not None:
        torch._check(lin_bias is not None, lambda: "lin_bias must be given with lin_weight")
        _check_fd(lin_weight, weight, "lin_weight")
        _check_fd(lin_bias, weight, "lin_bias")
    out, idx = _forward_outputs(x, weight, torch.float32)
    if relu and save_mask:
        mask = torch.empty((x.shape[0], x.shape[1], _mask_words(weight.shape[2])), dtype=torch.int32,
                           device=x.device)
    else:
        mask = torch.empty((0,), dtype=torch.int32, device=x.device)
    return out, idx, mask


@torch.library.register_fake("rtdl_num_embeddings_cuda::backward_epilogue")
def _backward_epilogue_fake(grad_output, x, bin_edges, inv_bin_widths, n_bins, weight, bin_indices, relu_mask,
                            lin_weight, relu, quant_dtype, compute_grad_x, compute_grad_weight,
                            compute_grad_bias, compute_grad_lin_weight, compute_grad_lin_bias):
    _check_backward_inputs(grad_output, x, weight, bin_indices)
    torch._check(grad_output.dtype == torch.float32, lambda: "grad_output must be float32")
    torch._check(quant_dtype in SUPPORTED_OUTPUT_DTYPES, lambda: "Unsupported quant dtype")
    if lin_weight is not None:
        _check_fd(lin_weight, weight, "lin_weight")
    torch._check(not (lin_weight is not None and compute_grad_bias),
                 lambda: "no bias gradient with lin_weight (version B has no bias)")
    torch._check(lin_weight is not None or not (compute_grad_lin_weight or compute_grad_lin_bias),
                 lambda: "linear0 gradients need lin_weight")
    if relu:
        torch._check(relu_mask.ndim == 3 and relu_mask.dtype == torch.int32,
                     lambda: "relu_mask must be the int32 [N, F, ceil(D / 32)] pass bits of the forward")

    def fd(wanted: bool) -> Tensor:
        shape = (weight.shape[0], weight.shape[2]) if wanted else (0,)
        return torch.empty(shape, dtype=weight.dtype, device=weight.device)

    return (_maybe(x, x, compute_grad_x), _maybe(weight, weight, compute_grad_weight), fd(compute_grad_bias),
            fd(compute_grad_lin_weight), fd(compute_grad_lin_bias))


@torch.library.register_fake("rtdl_num_embeddings_cuda::encode")
def _encode_fake(x, bin_edges, inv_bin_widths, n_bins, offsets, total_bins):
    torch._check(x.ndim == 2 and x.dtype == torch.float32, lambda: "x must be float32 [N, F]")
    torch._check(n_bins.shape[0] == x.shape[1], lambda: "n_bins must be int32 [F]")
    torch._check(offsets.shape[0] == x.shape[1], lambda: "offsets must be int32 [F]")
    torch._check(total_bins > 0, lambda: "total_bins must be positive")
    return torch.empty((x.shape[0], total_bins), dtype=torch.float32, device=x.device)


@torch.library.register_fake("rtdl_num_embeddings_cuda::encode_backward")
def _encode_backward_fake(grad_output, x, bin_edges, inv_bin_widths, n_bins, offsets):
    torch._check(grad_output.ndim == 2 and grad_output.shape[0] == x.shape[0],
                 lambda: "grad_output must be contiguous float32 [N, total_bins]")
    return torch.empty_like(x)


# ---------------------------------------------------------------------------
# lookup, residual norm, distillation loss
# ---------------------------------------------------------------------------

INDEX_DTYPES = (torch.int32, torch.int64)
NORM_MAX_WIDTH = 8192
DISTILL_STATS = 8


def _check_tokens(tokens, offsets) -> None:
    torch._check(tokens.dtype in INDEX_DTYPES, lambda: "tokens must be int32 or int64")
    if offsets is not None:
        torch._check(offsets.ndim == 1 and offsets.dtype == torch.int64, lambda: "offsets must be int64 [F + 1]")
        torch._check(tokens.ndim >= 1 and tokens.shape[-1] == offsets.shape[0] - 1,
                     lambda: "the last dimension of tokens must be offsets.size(0) - 1")


@torch.library.register_fake("rtdl_num_embeddings_cuda::lookup")
def _lookup_fake(tokens, weight, offsets, scale, padding_idx, output_dtype):
    _check_tokens(tokens, offsets)
    torch._check(weight.ndim == 2, lambda: "weight must have shape [V, D]")
    torch._check(weight.dtype in SUPPORTED_OUTPUT_DTYPES, lambda: "weight must be float32, float16, or bfloat16")
    torch._check(output_dtype in SUPPORTED_OUTPUT_DTYPES, lambda: "output_dtype must be float32, float16, or bfloat16")
    return weight.new_empty((*tokens.shape, weight.shape[1]), dtype=output_dtype)


@torch.library.register_fake("rtdl_num_embeddings_cuda::lookup_backward")
def _lookup_backward_fake(grad_output, tokens, offsets, num_rows, scale, padding_idx, grad_dtype):
    _check_tokens(tokens, offsets)
    torch._check(grad_output.ndim == tokens.ndim + 1,
                 lambda: "grad_output must have the shape of tokens and one more dimension")
    torch._check(grad_dtype in SUPPORTED_OUTPUT_DTYPES, lambda: "grad_dtype must be float32, float16, or bfloat16")
    return grad_output.new_empty((num_rows, grad_output.shape[-1]), dtype=grad_dtype)


@torch.library.register_fake("rtdl_num_embeddings_cuda::residual_norm")
def _residual_norm_fake(residual, branch, post_weight, post_bias, gate, pre_weight, pre_bias, post_norm, pre_norm,
                        gate_activation, residual_scale, eps, normed_dtype):
    torch._check(residual.ndim >= 1, lambda: "the residual stream must have shape [..., D]")
    torch._check(residual.dtype == torch.float32 or residual.dtype == normed_dtype,
                 lambda: "the residual stream must be float32 or of the branch's dtype")
    if branch is not None:
        torch._check(branch.dtype == normed_dtype, lambda: "normed_dtype must be the branch's dtype")
        torch._check(branch.shape == residual.shape, lambda: "branch must have the shape of the residual stream")
    else:
        torch._check(post_norm == 0 and gate is None and residual_scale == 1.0,
                     lambda: "without a branch there is no post norm, no gate and no residual scale")
        torch._check(pre_norm != 0, lambda: "without a branch there has to be a pre norm")
    d = residual.shape[-1]
    torch._check(d <= NORM_MAX_WIDTH, lambda: f"rows of at most {NORM_MAX_WIDTH} elements are supported, got {d}")
    for name, t in (("post_weight", post_weight), ("post_bias", post_bias), ("pre_weight", pre_weight),
                    ("pre_bias", pre_bias)):
        if t is not None:
            torch._check(t.ndim == 1 and t.shape[0] == d, lambda name=name: f"{name} must have shape [D]")
    if gate is not None:
        torch._check(gate.ndim == 2 and gate.shape[1] == d, lambda: "gate must have shape [G, D]")
    stream = torch.empty_like(residual) if branch is not None else residual.new_empty((0,))
    normed = (torch.empty_like(residual, dtype=normed_dtype) if pre_norm != 0
              else residual.new_empty((0,), dtype=normed_dtype))
    return stream, normed, residual.new_empty((residual.numel() // d, 4), dtype=torch.float32)


@torch.library.register_fake("rtdl_num_embeddings_cuda::residual_norm_backward")
def _residual_norm_backward_fake(grad_stream, grad_normed, stream, branch, stats, post_weight, post_bias, gate, pre_weight,
                                 pre_bias, post_norm, pre_norm, gate_activation, residual_scale, output_mask):
    if grad_stream is not None:
        torch._check(grad_stream.shape == stream.shape and grad_stream.dtype == stream.dtype,
                     lambda: "grad_stream must have the shape and dtype of stream")
    if grad_normed is not None:
        torch._check(pre_norm != 0, lambda: "grad_normed needs a pre norm")
        torch._check(grad_normed.shape == stream.shape,
                     lambda: "grad_normed must have the shape of stream and the branch's dtype")
    inputs = (stream, branch, post_weight, post_bias, gate, pre_weight, pre_bias)
    return tuple(torch.empty_like(t) if wanted and t is not None else stream.new_empty((0,))
                 for t, wanted in zip(inputs, output_mask))


def _check_distillation(logits, teacher_logits, teacher_classes, labels, temperature, alpha) -> None:
    torch._check(logits.ndim == 2, lambda: "logits must have shape [N, V]")
    torch._check(logits.dtype in SUPPORTED_OUTPUT_DTYPES, lambda: "logits must be float32, float16, or bfloat16")
    torch._check(teacher_logits.ndim == 2 and teacher_logits.shape[0] == logits.shape[0],
                 lambda: "teacher_logits must have shape [N, K]")
    torch._check(teacher_classes.shape == teacher_logits.shape, lambda: "teacher_classes must have shape [N, K]")
    torch._check(teacher_classes.dtype in INDEX_DTYPES, lambda: "teacher_classes must be int32 or int64")
    if labels is not None:
        torch._check(labels.ndim == 1 and labels.shape[0] == logits.shape[0] and labels.dtype == torch.int64,
                     lambda: "labels must be int64 [N]")
    torch._check(1e-6 < temperature < 1e6, lambda: f"temperature must be between 1e-6 and 1e6, got {temperature}")
    torch._check(0.0 <= alpha <= 1.0, lambda: f"alpha must be between 0 and 1, got {alpha}")


@torch.library.register_fake("rtdl_num_embeddings_cuda::distillation_loss")
def _distillation_loss_fake(logits, teacher_logits, teacher_classes, teacher_lse, labels, temperature, alpha):
    _check_distillation(logits, teacher_logits, teacher_classes, labels, temperature, alpha)
    n = logits.shape[0]
    return (logits.new_empty((n,), dtype=torch.float32), logits.new_empty((n, DISTILL_STATS), dtype=torch.float32))


@torch.library.register_fake("rtdl_num_embeddings_cuda::distillation_loss_backward")
def _distillation_loss_backward_fake(grad_loss, logits, teacher_logits, teacher_classes, labels, stats, temperature, alpha):
    _check_distillation(logits, teacher_logits, teacher_classes, labels, temperature, alpha)
    torch._check(grad_loss.ndim == 1 and grad_loss.dtype == torch.float32, lambda: "grad_loss must be float32 [N]")
    return torch.empty_like(logits)

"""ctypes binding of the C ABI in ``include/ple_hip.h`` (``libple_hip.so``).

This is the binding a caller without the torch operators would use: plain
device pointers, sizes, dtype codes and a stream handle.  The helpers below
take torch tensors only to read their pointers and sizes; nothing here copies
or allocates except :func:`backward`, which takes a workspace from the caller
or allocates one through torch.

Every entry point returns an ``int`` code; non-zero codes raise
:class:`PleError` with ``ple_error_string``'s text.
"""

from __future__ import annotations

import ctypes
import os

import torch

_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libple_hip.so")

DTYPE_F32, DTYPE_F16, DTYPE_BF16 = 0, 1, 2

# planner overrides (PLE_TUNE_* of the header; 0 = the planner's choice)
TUNE = {
    "FWD_FS": 0, "FWD_WG_PER_CU": 1, "FWD_FB": 2, "FWD_VEC": 3, "FWD_WIDE": 4, "BWD_SIMPLE": 5,
    "BWD_SIMPLE_GLOBAL": 6, "BWD_VEC": 7, "BWD_FS": 8, "BWD_RB": 9, "BWD_WG_PER_CU": 10, "BWD_MFMA": 11,
    "BWD_STREAM": 12, "GROUP_POLLS": 13,
}
_DTYPE_CODES = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16}

_lib = None


class Epilogue(ctypes.Structure):
    """``ple_epilogue_t``: the module tail fused into the kernels."""

    _fields_ = [
        ("bias", ctypes.c_void_p),
        ("lin_weight", ctypes.c_void_p),
        ("lin_bias", ctypes.c_void_p),
        ("relu", ctypes.c_int),
        ("relu_mask", ctypes.c_void_p),
    ]


class BackwardPlanInfo(ctypes.Structure):
    """``ple_backward_plan_info_t``: the backward's launch plan for a shape."""

    _fields_ = [
        ("sorted", ctypes.c_int),
        ("chunks", ctypes.c_int),
        ("features_per_group", ctypes.c_int),
        ("columns_per_lane", ctypes.c_int),
        ("lanes_per_row", ctypes.c_int),
        ("threads", ctypes.c_int),
        ("lds_bytes", ctypes.c_size_t),
        ("workspace_bytes", ctypes.c_size_t),
        ("bins_per_window", ctypes.c_int),
        ("windows", ctypes.c_int),
        ("matrix_cores", ctypes.c_int),
    ]


class EncodePlanInfo(ctypes.Structure):
    """``ple_encode_plan_info_t``: the dense encoding's launch plan for a shape."""

    _fields_ = [
        ("features_per_group", ctypes.c_int),
        ("features_searched", ctypes.c_int),
        ("groups", ctypes.c_int),
        ("chunks", ctypes.c_int),
        ("rows_per_block", ctypes.c_int),
        ("pairs_per_block", ctypes.c_int),
        ("lds_tables", ctypes.c_int),
        ("lds_bytes", ctypes.c_size_t),
    ]


class Grad(ctypes.Structure):
    """``ple_grad_t``: a gradient of a list, and where it goes when scaled."""

    _fields_ = [
        ("grad", ctypes.c_void_p),
        ("out", ctypes.c_void_p),
        ("numel", ctypes.c_int64),
        ("dtype", ctypes.c_int),
        ("out_dtype", ctypes.c_int),
    ]


class LookupPlanInfo(ctypes.Structure):
    """``ple_lookup_plan_info_t``: the lookup backward's launch plan for a shape."""

    _fields_ = [
        ("one_workgroup", ctypes.c_int),
        ("passes", ctypes.c_int),
        ("digit_bits", ctypes.c_int),
        ("sort_workgroups", ctypes.c_int),
        ("sum_workgroups", ctypes.c_int64),
        ("clear_rows", ctypes.c_int64),
        ("most_threads", ctypes.c_int64),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class GroupNormPlanInfo(ctypes.Structure):
    """``ple_group_norm_plan_info_t``: the group norm's launch plan for a shape."""

    _fields_ = [
        ("form", ctypes.c_int),
        ("lane_channels", ctypes.c_int),
        ("slabs", ctypes.c_int),
        ("members", ctypes.c_int),
        ("params_end", ctypes.c_int64),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class Norm(ctypes.Structure):
    """``ple_norm_t``: the norms, gate and residual scale around a block."""

    _fields_ = [
        ("post_weight", ctypes.c_void_p),
        ("post_bias", ctypes.c_void_p),
        ("gate", ctypes.c_void_p),
        ("pre_weight", ctypes.c_void_p),
        ("pre_bias", ctypes.c_void_p),
        ("gate_rows", ctypes.c_int64),
        ("post_norm", ctypes.c_int),
        ("pre_norm", ctypes.c_int),
        ("gate_activation", ctypes.c_int),
        ("stream_dtype", ctypes.c_int),
        ("branch_dtype", ctypes.c_int),
        ("param_dtype", ctypes.c_int),
        ("residual_scale", ctypes.c_float),
        ("eps", ctypes.c_float),
    ]


class NormGrads(ctypes.Structure):
    """``ple_norm_grads_t``: the gradients a norm's backward writes."""

    _fields_ = [
        ("residual", ctypes.c_void_p),
        ("branch", ctypes.c_void_p),
        ("post_weight", ctypes.c_void_p),
        ("post_bias", ctypes.c_void_p),
        ("gate", ctypes.c_void_p),
        ("pre_weight", ctypes.c_void_p),
        ("pre_bias", ctypes.c_void_p),
    ]


class PleError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"{message} (code {code})")
        self.code = code


def lib() -> ctypes.CDLL:
    """Loads ``libple_hip.so`` once and declares every prototype."""
    global _lib
    if _lib is None:
        if not os.path.exists(_LIB_PATH):
            raise RuntimeError(f"{_LIB_PATH} is not built; run piecewiselinearembeddings_optimized_amd._build")
        L = ctypes.CDLL(_LIB_PATH)
        p, i64, i32, sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t
        L.ple_abi_version.argtypes, L.ple_abi_version.restype = [], i32
        L.ple_bin_index_bytes.argtypes, L.ple_bin_index_bytes.restype = [i64], i32
        L.ple_error_string.argtypes, L.ple_error_string.restype = [i32], ctypes.c_char_p
        L.ple_set_tuning.argtypes, L.ple_set_tuning.restype = [i32, i32], i32
        L.ple_forward_launch.argtypes = [p, p, p, p, p, p, p, p, i64, i64, i64, i64, i32, i32, p]
        L.ple_forward_launch.restype = i32
        L.ple_backward_workspace_bytes.argtypes = [i64, i64, i64, i64]
        L.ple_backward_workspace_bytes.restype = sz
        L.ple_backward_launch.argtypes = [p, p, p, p, p, p, p, p, p, p, i64, i64, i64, i64, i32, i32, p, sz, p]
        L.ple_backward_launch.restype = i32
        L.ple_backward_launch_noalloc.argtypes = [p, p, p, p, p, p, p, p, p, p, i64, i64, i64, i64, i32, i32, p]
        L.ple_backward_launch_noalloc.restype = i32
        L.ple_backward_plan_query.argtypes = [p, i64, i64, i64, i64, i32, i32, i32, i32,
                                              ctypes.POINTER(BackwardPlanInfo)]
        L.ple_backward_plan_query.restype = i32
        ep = ctypes.POINTER(Epilogue)
        L.ple_forward_epilogue_launch.argtypes = [p, p, p, p, p, ep, p, p, i64, i64, i64, i64, i32, p]
        L.ple_forward_epilogue_launch.restype = i32
        L.ple_backward_epilogue_launch.argtypes = [p, p, p, p, p, p, p, ep, p, p, p, p, p, i64, i64, i64, i64, i32,
                                                   p, sz, p]
        L.ple_backward_epilogue_launch.restype = i32
        L.ple_encode_launch.argtypes = [p, p, p, p, p, p, i64, i64, i64, i64, p]
        L.ple_encode_launch.restype = i32
        L.ple_encode_backward_launch.argtypes = [p, p, p, p, p, p, p, i64, i64, i64, i64, p]
        L.ple_encode_backward_launch.restype = i32
        L.ple_encode_plan_query.argtypes = [p, i64, i64, i64, i64, i32, ctypes.POINTER(EncodePlanInfo)]
        L.ple_encode_plan_query.restype = i32
        f32, np_, gp = ctypes.c_float, ctypes.POINTER(Norm), ctypes.POINTER(NormGrads)
        L.ple_lookup_launch.argtypes = [p, i32, p, p, p, i64, i64, i64, i64, f32, i32, i32, p]
        L.ple_lookup_launch.restype = i32
        L.ple_lookup_backward_workspace_bytes.argtypes = [i64, i64, i64]
        L.ple_lookup_backward_workspace_bytes.restype = sz
        L.ple_lookup_backward_launch.argtypes = [p, p, i32, p, p, i64, i64, i64, i64, i64, f32, i32, i32, p, sz, p]
        L.ple_lookup_backward_launch.restype = i32
        L.ple_lookup_backward_plan_query.argtypes = [p, p, i64, i64, i64, i32, i32, ctypes.POINTER(LookupPlanInfo)]
        L.ple_lookup_backward_plan_query.restype = i32
        L.ple_residual_norm_launch.argtypes = [p, p, np_, p, p, p, i64, i64, p]
        L.ple_residual_norm_launch.restype = i32
        L.ple_residual_norm_backward_workspace_bytes.argtypes = [np_, i64, i64]
        L.ple_residual_norm_backward_workspace_bytes.restype = sz
        L.ple_residual_norm_backward_launch.argtypes = [p, p, p, p, p, np_, gp, i64, i64, p, sz, p]
        L.ple_residual_norm_backward_launch.restype = i32
        L.ple_distill_workspace_bytes.argtypes, L.ple_distill_workspace_bytes.restype = [i64, i64], sz
        L.ple_distill_launch.argtypes = [p, p, p, i32, p, p, p, p, i64, i64, i64, f32, f32, i32, i32, p, sz, p]
        L.ple_distill_launch.restype = i32
        L.ple_distill_backward_launch.argtypes = [p, p, p, p, i32, p, p, p, i64, i64, i64, f32, f32, i32, i32, p]
        L.ple_distill_backward_launch.restype = i32
        L.ple_group_norm_workspace_bytes.argtypes = [i64, i64, i64, i64, i32]
        L.ple_group_norm_workspace_bytes.restype = sz
        L.ple_group_norm_launch.argtypes = [p, p, p, p, p, i64, i64, i64, i64, i32, f32, i32, i32, p, sz, p]
        L.ple_group_norm_launch.restype = i32
        L.ple_group_norm_backward_workspace_bytes.argtypes = [i64, i64, i64, i64, i32]
        L.ple_group_norm_backward_workspace_bytes.restype = sz
        L.ple_group_norm_backward_launch.argtypes = [p, p, p, p, p, p, p, p, i64, i64, i64, i64, i32, i32, i32, p, sz, p]
        L.ple_group_norm_backward_launch.restype = i32
        L.ple_group_norm_plan_query.argtypes = [p, i64, i64, i64, i64, i32, i32, ctypes.POINTER(GroupNormPlanInfo)]
        L.ple_group_norm_plan_query.restype = i32
        L.ple_relative_bias_launch.argtypes = [p, p, p, p, i64, i64, i64, i64, i64, i64, i64, i32, i32, i32, p]
        L.ple_relative_bias_launch.restype = i32
        L.ple_relative_bias_backward_workspace_bytes.argtypes = [i64, i64, i64, i64, i64, i64]
        L.ple_relative_bias_backward_workspace_bytes.restype = sz
        L.ple_relative_bias_backward_launch.argtypes = [p, p, p, p, i64, i64, i64, i64, i64, i64, i64, i32, i32, i32, p, sz, p]
        L.ple_relative_bias_backward_launch.restype = i32
        L.ple_grad_norm_workspace_bytes.argtypes = [ctypes.POINTER(Grad), i64]
        L.ple_grad_norm_workspace_bytes.restype = sz
        L.ple_grad_norm_launch.argtypes = [ctypes.POINTER(Grad), i64, i32, p, p, sz, p]
        L.ple_grad_norm_launch.restype = i32
        L.ple_grad_scale_launch.argtypes = [ctypes.POINTER(Grad), i64, p, f32, p]
        L.ple_grad_scale_launch.restype = i32
        L.ple_grad_clip_launch.argtypes = [ctypes.POINTER(Grad), i64, i32, f32, p, p, sz, p]
        L.ple_grad_clip_launch.restype = i32
        L.ple_timing_start.argtypes, L.ple_timing_start.restype = [i32], i32
        L.ple_timing_stop.argtypes, L.ple_timing_stop.restype = [], i32
        L.ple_timing_read.argtypes = [i32, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_int)]
        L.ple_timing_read.restype = i32
        _lib = L
    return _lib


def set_tuning(knob: str, value: int) -> int:
    """Sets planner override ``knob`` (a key of :data:`TUNE`); returns the
    previous value.  0 restores the planner's own choice."""
    return lib().ple_set_tuning(TUNE[knob], int(value))


TIMER_FORWARD, TIMER_BACKWARD = 0, 1


def timing_start(slots: int) -> None:
    """``ple_timing_start``: time the main kernel of the next ``slots``
    forward and backward launches (0 releases the events)."""
    check(lib().ple_timing_start(int(slots)))


def timing_stop() -> None:
    check(lib().ple_timing_stop())


def timing_read(which: int):
    """``(total_ms, launches)`` recorded for ``TIMER_FORWARD`` / ``TIMER_BACKWARD``."""
    ms = ctypes.c_double(0.0)
    n = ctypes.c_int(0)
    check(lib().ple_timing_read(int(which), ctypes.byref(ms), ctypes.byref(n)))
    return ms.value, n.value


def check(code: int) -> None:
    if code != 0:
        raise PleError(code, lib().ple_error_string(code).decode())


def dtype_code(dtype: torch.dtype) -> int:
    return _DTYPE_CODES[dtype]


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(stream):
    if stream is None:
        stream = torch.cuda.current_stream()
    return ctypes.c_void_p(stream.cuda_stream)


def forward(x, bin_edges, inv_bin_widths, n_bins, weight, bias, output, bin_indices, quant_dtype,
            stream=None) -> None:
    """``ple_forward_launch`` into caller-provided ``output`` / ``bin_indices``."""
    n, f = x.shape
    _, bmax, d = weight.shape
    check(lib().ple_forward_launch(
        _ptr(x), _ptr(bin_edges), _ptr(inv_bin_widths), _ptr(n_bins), _ptr(weight), _ptr(bias),
        _ptr(output), _ptr(bin_indices), n, f, bmax, d, dtype_code(quant_dtype), dtype_code(output.dtype),
        _stream(stream)))


def workspace_bytes(n: int, f: int, bmax: int, d: int) -> int:
    return int(lib().ple_backward_workspace_bytes(n, f, bmax, d))


def backward_plan(n: int, f: int, bmax: int, d: int, grad_dtype=torch.float32, quant_dtype=None,
                  relu: bool = False, linear0: bool = False, grad_output=None) -> dict:
    """``ple_backward_plan_query``: the plan a backward launch of this shape
    takes, as a dict of :class:`BackwardPlanInfo`'s fields."""
    info = BackwardPlanInfo()
    q = grad_dtype if quant_dtype is None else quant_dtype
    check(lib().ple_backward_plan_query(_ptr(grad_output), n, f, bmax, d, dtype_code(grad_dtype), dtype_code(q),
                                        1 if relu else 0, 1 if linear0 else 0, ctypes.byref(info)))
    return {name: getattr(info, name) for name, _ in BackwardPlanInfo._fields_}


def encode_plan(n: int, f: int, bmax: int, total_bins: int, backward: bool = False, output=None) -> dict:
    """``ple_encode_plan_query``: the plan an encoding (or its backward) of
    this shape takes, as a dict of :class:`EncodePlanInfo`'s fields."""
    info = EncodePlanInfo()
    check(lib().ple_encode_plan_query(_ptr(output), n, f, bmax, total_bins, 1 if backward else 0, ctypes.byref(info)))
    return {name: getattr(info, name) for name, _ in EncodePlanInfo._fields_}


def backward(grad_output, x, bin_edges, inv_bin_widths, n_bins, weight, bin_indices, grad_x, grad_weight,
             grad_bias, quant_dtype, workspace=None, stream=None) -> None:
    """``ple_backward_launch``; ``grad_*`` are caller-provided fp32 tensors or None."""
    n, f = x.shape
    _, bmax, d = weight.shape
    need = workspace_bytes(n, f, bmax, d)
    if workspace is None and need > 0:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    check(lib().ple_backward_launch(
        _ptr(grad_output), _ptr(x), _ptr(bin_edges), _ptr(inv_bin_widths), _ptr(n_bins), _ptr(weight),
        _ptr(bin_indices), _ptr(grad_x), _ptr(grad_weight), _ptr(grad_bias), n, f, bmax, d,
        dtype_code(grad_output.dtype), dtype_code(quant_dtype), _ptr(workspace), ws_bytes, _stream(stream)))


def epilogue(bias=None, lin_weight=None, lin_bias=None, relu=False, relu_mask=None) -> Epilogue:
    def addr(t):
        return None if t is None else t.data_ptr()

    return Epilogue(addr(bias), addr(lin_weight), addr(lin_bias), 1 if relu else 0, addr(relu_mask))


def forward_epilogue(x, bin_edges, inv_bin_widths, n_bins, weight, epi: Epilogue, output, bin_indices,
                     quant_dtype, stream=None) -> None:
    """``ple_forward_epilogue_launch`` (fp32 ``output``)."""
    n, f = x.shape
    _, bmax, d = weight.shape
    check(lib().ple_forward_epilogue_launch(
        _ptr(x), _ptr(bin_edges), _ptr(inv_bin_widths), _ptr(n_bins), _ptr(weight), ctypes.byref(epi),
        _ptr(output), _ptr(bin_indices), n, f, bmax, d, dtype_code(quant_dtype), _stream(stream)))


def backward_epilogue(grad_output, x, bin_edges, inv_bin_widths, n_bins, weight, bin_indices, epi: Epilogue,
                      grad_x, grad_weight, grad_bias, grad_lin_weight, grad_lin_bias, quant_dtype,
                      workspace=None, stream=None) -> None:
    """``ple_backward_epilogue_launch``; gradients are caller-provided fp32 tensors or None."""
    n, f = x.shape
    _, bmax, d = weight.shape
    need = workspace_bytes(n, f, bmax, d)
    if workspace is None and need > 0:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    ws_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    check(lib().ple_backward_epilogue_launch(
        _ptr(grad_output), _ptr(x), _ptr(bin_edges), _ptr(inv_bin_widths), _ptr(n_bins), _ptr(weight),
        _ptr(bin_indices), ctypes.byref(epi), _ptr(grad_x), _ptr(grad_weight), _ptr(grad_bias),
        _ptr(grad_lin_weight), _ptr(grad_lin_bias), n, f, bmax, d, dtype_code(quant_dtype), _ptr(workspace),
        ws_bytes, _stream(stream)))


def encode(x, bin_edges, inv_bin_widths, n_bins, offsets, output, stream=None) -> None:
    """``ple_encode_launch`` into a caller-provided fp32 ``output`` [N, total_bins]."""
    n, f = x.shape
    check(lib().ple_encode_launch(
        _ptr(x), _ptr(bin_edges), _ptr(inv_bin_widths), _ptr(n_bins), _ptr(offsets), _ptr(output), n, f,
        inv_bin_widths.shape[1], output.shape[1], _stream(stream)))


def encode_backward(grad_output, x, bin_edges, inv_bin_widths, n_bins, offsets, grad_x, stream=None) -> None:
    """``ple_encode_backward_launch`` into a caller-provided fp32 ``grad_x`` [N, F]."""
    n, f = x.shape
    check(lib().ple_encode_backward_launch(
        _ptr(grad_output), _ptr(x), _ptr(bin_edges), _ptr(inv_bin_widths), _ptr(n_bins), _ptr(offsets),
        _ptr(grad_x), n, f, inv_bin_widths.shape[1], grad_output.shape[1], _stream(stream)))


def _workspace(need: int, like):
    return (torch.empty(need, dtype=torch.uint8, device=like.device) if need > 0 else None), need


def lookup(tokens, weight, output, offsets=None, scale=1.0, stream=None) -> None:
    """``ple_lookup_launch`` into a caller-provided ``output`` [*tokens.shape, D]."""
    v, d = weight.shape
    check(lib().ple_lookup_launch(
        _ptr(tokens), tokens.element_size(), _ptr(offsets), _ptr(weight), _ptr(output), tokens.numel(),
        1 if offsets is None else offsets.numel() - 1, v, d, scale, dtype_code(weight.dtype), dtype_code(output.dtype),
        _stream(stream)))


def lookup_backward(grad_output, tokens, grad_weight, offsets=None, scale=1.0, padding_idx=-1, workspace=None,
                    stream=None) -> None:
    """``ple_lookup_backward_launch`` into a caller-provided ``grad_weight`` [V, D]."""
    v, d = grad_weight.shape
    need = int(lib().ple_lookup_backward_workspace_bytes(tokens.numel(), v, d))
    if workspace is None:
        workspace, need = _workspace(need, tokens)
    else:
        need = workspace.numel() * workspace.element_size()
    check(lib().ple_lookup_backward_launch(
        _ptr(grad_output), _ptr(tokens), tokens.element_size(), _ptr(offsets), _ptr(grad_weight), tokens.numel(),
        1 if offsets is None else offsets.numel() - 1, v, d, padding_idx, scale, dtype_code(grad_output.dtype),
        dtype_code(grad_weight.dtype), _ptr(workspace), need, _stream(stream)))


def lookup_backward_plan(t: int, v: int, d: int, grad_dtype=torch.float32, weight_dtype=None, grad_output=None,
                         grad_weight=None) -> dict:
    """``ple_lookup_backward_plan_query``: the plan a gradient of ``t`` tokens'
    rows of a table [v, d] takes, as a dict of :class:`LookupPlanInfo`'s fields."""
    info = LookupPlanInfo()
    check(lib().ple_lookup_backward_plan_query(_ptr(grad_output), _ptr(grad_weight), t, v, d, dtype_code(grad_dtype),
                                               dtype_code(grad_dtype if weight_dtype is None else weight_dtype),
                                               ctypes.byref(info)))
    return {name: getattr(info, name) for name, _ in LookupPlanInfo._fields_}


def norm(stream_dtype, branch_dtype, post_norm=0, pre_norm=0, post_weight=None, post_bias=None, gate=None,
         gate_activation=0, pre_weight=None, pre_bias=None, residual_scale=1.0, eps=1e-5) -> Norm:
    """The descriptor of a residual norm (the tensors have to outlive it)."""
    def addr(t):
        return None if t is None else t.data_ptr()

    given = [t for t in (post_weight, post_bias, gate, pre_weight, pre_bias) if t is not None]
    return Norm(addr(post_weight), addr(post_bias), addr(gate), addr(pre_weight), addr(pre_bias),
                0 if gate is None else gate.shape[0], post_norm, pre_norm, gate_activation, dtype_code(stream_dtype),
                dtype_code(branch_dtype), dtype_code(given[0].dtype) if given else DTYPE_F32, residual_scale, eps)


def residual_norm(residual, branch, descriptor: Norm, stream_out, normed, stats, stream=None) -> None:
    """``ple_residual_norm_launch`` into caller-provided outputs."""
    n, d = residual.shape
    check(lib().ple_residual_norm_launch(_ptr(residual), _ptr(branch), ctypes.byref(descriptor), _ptr(stream_out),
                                         _ptr(normed), _ptr(stats), n, d, _stream(stream)))


def residual_norm_backward(grad_stream, grad_normed, stream_in, branch, stats, descriptor: Norm, grads: dict,
                           workspace=None, stream=None) -> None:
    """``ple_residual_norm_backward_launch``; ``grads``: caller-provided tensors
    by :class:`NormGrads`'s field names."""
    n, d = stream_in.shape
    if workspace is None:
        workspace, need = _workspace(
            int(lib().ple_residual_norm_backward_workspace_bytes(ctypes.byref(descriptor), n, d)), stream_in)
    else:
        need = workspace.numel() * workspace.element_size()
    out = NormGrads(**{k: t.data_ptr() for k, t in grads.items() if t is not None})
    check(lib().ple_residual_norm_backward_launch(
        _ptr(grad_stream), _ptr(grad_normed), _ptr(stream_in), _ptr(branch), _ptr(stats), ctypes.byref(descriptor),
        ctypes.byref(out), n, d, _ptr(workspace), need, _stream(stream)))


def distill(logits, teacher_logits, teacher_classes, loss, stats, teacher_lse=None, labels=None, temperature=1.0,
            alpha=1.0, workspace=None, stream=None) -> None:
    """``ple_distill_launch`` into caller-provided ``loss`` [N] and ``stats`` [N, 8]."""
    n, v = logits.shape
    if workspace is None:
        workspace, need = _workspace(int(lib().ple_distill_workspace_bytes(n, v)), logits)
    else:
        need = workspace.numel() * workspace.element_size()
    check(lib().ple_distill_launch(
        _ptr(logits), _ptr(teacher_logits), _ptr(teacher_classes), teacher_classes.element_size(), _ptr(teacher_lse),
        _ptr(labels), _ptr(loss), _ptr(stats), n, v, teacher_logits.shape[1], temperature, alpha,
        dtype_code(logits.dtype), dtype_code(teacher_logits.dtype), _ptr(workspace), need, _stream(stream)))


def distill_backward(grad_loss, logits, teacher_logits, teacher_classes, stats, grad_logits, labels=None,
                     temperature=1.0, alpha=1.0, stream=None) -> None:
    """``ple_distill_backward_launch`` into a caller-provided ``grad_logits`` [N, V]."""
    n, v = logits.shape
    check(lib().ple_distill_backward_launch(
        _ptr(grad_loss), _ptr(logits), _ptr(teacher_logits), _ptr(teacher_classes), teacher_classes.element_size(),
        _ptr(labels), _ptr(stats), _ptr(grad_logits), n, v, teacher_logits.shape[1], temperature, alpha,
        dtype_code(logits.dtype), dtype_code(teacher_logits.dtype), _stream(stream)))


def group_norm(x, weight, bias, y, stats, num_groups, activation=0, eps=1e-5, workspace=None, stream=None) -> None:
    """``ple_group_norm_launch`` into caller-provided ``y`` (as ``x`` [N, S, C]) and ``stats`` [N, G, 2]."""
    n, s, c = x.shape
    param = next((t.dtype for t in (weight, bias) if t is not None), torch.float32)
    if workspace is None:
        workspace, need = _workspace(int(lib().ple_group_norm_workspace_bytes(n, s, c, num_groups, dtype_code(x.dtype))), x)
    else:
        need = workspace.numel() * workspace.element_size()
    check(lib().ple_group_norm_launch(
        _ptr(x), _ptr(weight), _ptr(bias), _ptr(y), _ptr(stats), n, s, c, num_groups, activation, eps, dtype_code(x.dtype),
        dtype_code(param), _ptr(workspace), need, _stream(stream)))


def group_norm_backward(grad_y, x, stats, weight, bias, grad_x, grad_weight, grad_bias, num_groups, activation=0,
                        workspace=None, stream=None) -> None:
    """``ple_group_norm_backward_launch``; gradients are caller-provided tensors or None."""
    n, s, c = x.shape
    param = next((t.dtype for t in (weight, bias) if t is not None), torch.float32)
    if workspace is None:
        workspace, need = _workspace(
            int(lib().ple_group_norm_backward_workspace_bytes(n, s, c, num_groups, dtype_code(x.dtype))), x)
    else:
        need = workspace.numel() * workspace.element_size()
    check(lib().ple_group_norm_backward_launch(
        _ptr(grad_y), _ptr(x), _ptr(stats), _ptr(weight), _ptr(bias), _ptr(grad_x), _ptr(grad_weight), _ptr(grad_bias), n, s,
        c, num_groups, activation, dtype_code(x.dtype), dtype_code(param), _ptr(workspace), need, _stream(stream)))


def group_norm_plan(n, s, c, num_groups, dtype=torch.float32, backward=False, x=None) -> dict:
    """The launch plan for samples [n, s, c] (``x``: a tensor whose alignment counts), as a dict of
    :class:`GroupNormPlanInfo`'s fields."""
    info = GroupNormPlanInfo()
    check(lib().ple_group_norm_plan_query(_ptr(x), n, s, c, num_groups, dtype_code(dtype), int(backward), ctypes.byref(info)))
    return {name: getattr(info, name) for name, _ in GroupNormPlanInfo._fields_}


def relative_bias(weight, buckets, out, starts=None, offset=0, causal=False, stream=None) -> None:
    """``ple_relative_bias_launch`` into a caller-provided ``out`` [H, q, k] ([B, H, q, k] with ``starts``)."""
    r, h = weight.shape
    check(lib().ple_relative_bias_launch(
        _ptr(weight), _ptr(buckets), _ptr(starts), _ptr(out), 1 if starts is None else starts.numel(), h, out.shape[-2],
        out.shape[-1], r, buckets.numel() // 2, offset, int(causal), dtype_code(weight.dtype), dtype_code(out.dtype),
        _stream(stream)))


def relative_bias_backward(grad_output, buckets, grad_weight, starts=None, offset=0, causal=False, workspace=None,
                           stream=None) -> None:
    """``ple_relative_bias_backward_launch`` into a caller-provided ``grad_weight`` [R, H]."""
    r, h = grad_weight.shape
    b, q, k, far = 1 if starts is None else starts.numel(), *grad_output.shape[-2:], buckets.numel() // 2
    if workspace is None:
        workspace, need = _workspace(int(lib().ple_relative_bias_backward_workspace_bytes(b, h, q, k, r, far)), grad_output)
    else:
        need = workspace.numel() * workspace.element_size()
    check(lib().ple_relative_bias_backward_launch(
        _ptr(grad_output), _ptr(buckets), _ptr(starts), _ptr(grad_weight), b, h, q, k, r, far, offset, int(causal),
        dtype_code(grad_output.dtype), dtype_code(grad_weight.dtype), _ptr(workspace), need, _stream(stream)))


def gradient_list(grads, out=None):
    """The host array of ``ple_grad_t`` of tensors that are contiguous (``out``: where they go; in place without)."""
    pairs = list(zip(grads, grads if out is None else out))
    return (Grad * len(pairs))(*(Grad(g.data_ptr(), o.data_ptr(), g.numel(), dtype_code(g.dtype), dtype_code(o.dtype))
                                 for g, o in pairs)), len(pairs)


def grad_norm(grads, norm, kind=2, workspace=None, stream=None) -> None:
    """``ple_grad_norm_launch`` (``kind``: 1, 2, or 3 for the largest) into a caller-provided float32 ``norm``."""
    listed, count = gradient_list(grads)
    if workspace is None:
        workspace, need = _workspace(int(lib().ple_grad_norm_workspace_bytes(listed, count)), norm)
    else:
        need = workspace.numel() * workspace.element_size()
    check(lib().ple_grad_norm_launch(listed, count, kind, _ptr(norm), _ptr(workspace), need, _stream(stream)))


def grad_scale(grads, norm, limit, out=None, stream=None) -> None:
    """``ple_grad_scale_launch``: in place, or into ``out``."""
    listed, count = gradient_list(grads, out)
    check(lib().ple_grad_scale_launch(listed, count, _ptr(norm), limit, _stream(stream)))


def grad_clip(grads, norm, limit, kind=2, out=None, workspace=None, stream=None) -> None:
    """``ple_grad_clip_launch``: :func:`grad_norm` into ``norm``, and :func:`grad_scale` with it."""
    listed, count = gradient_list(grads, out)
    if workspace is None:
        workspace, need = _workspace(int(lib().ple_grad_norm_workspace_bytes(listed, count)), norm)
    else:
        need = workspace.numel() * workspace.element_size()
    check(lib().ple_grad_clip_launch(listed, count, kind, limit, _ptr(norm), _ptr(workspace), need, _stream(stream)))

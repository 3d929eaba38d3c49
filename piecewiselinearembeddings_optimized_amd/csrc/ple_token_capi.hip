// The extern "C" entry points of the operators around the embedding (lookup,
// residual norm, distillation loss): argument checks that need no device, then
// the launchers.

#include "ple_internal.h"

namespace ple {
namespace {

// (token positions and sort keys are 32-bit; so are a row's vectors)
constexpr int64_t kMaxTokens = INT32_MAX - 1;
constexpr int64_t kMaxRows = INT32_MAX - 1;
constexpr int64_t kMaxWidth = 1 << 20;

int check_lookup(int64_t T, int64_t F, int64_t V, int64_t D, bool columns) {
    if (T < 0 || V < 1 || D < 1 || F < 1 || (columns && T % F != 0)) return PLE_E_BAD_SHAPE;
    if (T > kMaxTokens || V > kMaxRows || D > kMaxWidth || F > kMaxRows) return PLE_E_TOO_LARGE;
    return PLE_OK;
}

int check_token_bytes(int bytes) { return bytes == 4 || bytes == 8 ? PLE_OK : PLE_E_BAD_INDEX_WIDTH; }

bool valid_norm(int k) { return k == PLE_NORM_NONE || k == PLE_NORM_RMS || k == PLE_NORM_LAYER; }

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

bool aligned_for(const void *p, int dtype) { return aligned(p, dtype == PLE_DTYPE_F32 ? 4 : 2); }

// Shapes, types and pairings; `rows` are checked where there are rows.
int check_norm(const ple_norm_t *d, int64_t N, int64_t D) {
    if (!d) return PLE_E_NULL_POINTER;
    if (N < 0 || D < 1) return PLE_E_BAD_SHAPE;
    if (D > PLE_NORM_MAX_WIDTH || N > INT64_MAX / D / 8) return PLE_E_TOO_LARGE;
    if (!valid_dtype(d->stream_dtype) || !valid_dtype(d->branch_dtype) || !valid_dtype(d->param_dtype)) return PLE_E_BAD_DTYPE;
    if (d->stream_dtype != PLE_DTYPE_F32 && d->stream_dtype != d->branch_dtype) return PLE_E_UNSUPPORTED;
    if (!valid_norm(d->post_norm) || !valid_norm(d->pre_norm) || d->gate_activation < PLE_GATE_IDENTITY ||
        d->gate_activation > PLE_GATE_TANH)
        return PLE_E_UNSUPPORTED;
    if (d->post_norm == PLE_NORM_NONE && (d->post_weight || d->post_bias)) return PLE_E_UNSUPPORTED;
    if (d->pre_norm == PLE_NORM_NONE && (d->pre_weight || d->pre_bias)) return PLE_E_UNSUPPORTED;
    if (d->gate && (d->gate_rows < 1 || (N > 0 && (d->gate_rows > N || N % d->gate_rows != 0)))) return PLE_E_BAD_SHAPE;
    for (const void *p : {d->post_weight, d->post_bias, d->gate, d->pre_weight, d->pre_bias})
        if (!aligned_for(p, d->param_dtype)) return PLE_E_MISALIGNED;
    return PLE_OK;
}

NormRequest norm_request(const ple_norm_t *d, int64_t N, int64_t D, void *stream) {
    NormRequest r{};
    r.post_w = d->post_weight; r.post_b = d->post_bias; r.gate = d->gate;
    r.pre_w = d->pre_weight; r.pre_b = d->pre_bias;
    r.groups = d->gate ? d->gate_rows : 0;
    r.N = N; r.D = D;
    r.stream_dtype = d->stream_dtype; r.branch_dtype = d->branch_dtype; r.param_dtype = d->param_dtype;
    r.post = d->post_norm; r.pre = d->pre_norm; r.act = d->gate_activation;
    r.alpha = d->residual_scale; r.eps = d->eps;
    r.stream = static_cast<hipStream_t>(stream);
    return r;
}

int check_distill(int64_t N, int64_t V, int64_t K, int dtype, int teacher_dtype, int class_bytes, float temperature,
                  float alpha) {
    if (N < 0 || V < 1 || K < 1) return PLE_E_BAD_SHAPE;
    if (!valid_dtype(dtype) || !valid_dtype(teacher_dtype)) return PLE_E_BAD_DTYPE;
    if (class_bytes != 4 && class_bytes != 8) return PLE_E_BAD_INDEX_WIDTH;
    if (V > (int64_t{1} << 30) || K > (int64_t{1} << 20) || N > (int64_t{1} << 40) / V || N > (1 << 24)) return PLE_E_TOO_LARGE;
    // (written so that a NaN fails)
    if (!(temperature > 0.0f && temperature < 1e6f && temperature > 1e-6f) || !(alpha >= 0.0f && alpha <= 1.0f))
        return PLE_E_UNSUPPORTED;
    return PLE_OK;
}

}  // namespace
}  // namespace ple

extern "C" {

int ple_lookup_launch(const void *tokens, int token_bytes, const int64_t *offsets, const void *weight, void *output,
                      int64_t T, int64_t F, int64_t V, int64_t D, float scale, int weight_dtype, int output_dtype,
                      void *stream) {
    int rc = ple::check_lookup(T, F, V, D, offsets != nullptr);
    if (rc == PLE_OK) rc = ple::check_token_bytes(token_bytes);
    if (rc != PLE_OK) return rc;
    if (!ple::valid_dtype(weight_dtype) || !ple::valid_dtype(output_dtype)) return PLE_E_BAD_DTYPE;
    if (T == 0) return PLE_OK;
    if (!tokens || !weight || !output) return PLE_E_NULL_POINTER;
    if (!ple::aligned(tokens, token_bytes) || !ple::aligned(offsets, 8) || !ple::aligned_for(weight, weight_dtype) ||
        !ple::aligned_for(output, output_dtype))
        return PLE_E_MISALIGNED;
    ple::LookupRequest r{};
    r.tokens = tokens; r.offsets = offsets; r.table = weight; r.out = output;
    r.T = T; r.F = F; r.V = V; r.D = D;
    r.wide = token_bytes == 8; r.table_dtype = weight_dtype; r.out_dtype = output_dtype;
    r.scale = scale;
    r.stream = static_cast<hipStream_t>(stream);
    return ple::lookup_run(r);
}

size_t ple_lookup_backward_workspace_bytes(int64_t T, int64_t V, int64_t D) {
    return ple::check_lookup(T, 1, V, D, false) == PLE_OK ? ple::lookup_backward_workspace_bytes(T, V, D) : 0;
}

int ple_lookup_backward_launch(const void *grad_output, const void *tokens, int token_bytes, const int64_t *offsets,
                               void *grad_weight, int64_t T, int64_t F, int64_t V, int64_t D, int64_t padding_idx,
                               float scale, int grad_dtype, int weight_dtype, void *workspace, size_t workspace_bytes,
                               void *stream) {
    int rc = ple::check_lookup(T, F, V, D, offsets != nullptr);
    if (rc == PLE_OK) rc = ple::check_token_bytes(token_bytes);
    if (rc != PLE_OK) return rc;
    if (!ple::valid_dtype(grad_dtype) || !ple::valid_dtype(weight_dtype)) return PLE_E_BAD_DTYPE;
    if (!grad_weight || (T > 0 && (!grad_output || !tokens))) return PLE_E_NULL_POINTER;
    if (!ple::aligned(tokens, token_bytes) || !ple::aligned(offsets, 8) || !ple::aligned_for(grad_output, grad_dtype) ||
        !ple::aligned_for(grad_weight, weight_dtype))
        return PLE_E_MISALIGNED;
    ple::LookupRequest r{};
    r.tokens = tokens; r.offsets = offsets; r.grad = grad_output; r.dw = grad_weight;
    r.T = T; r.F = F; r.V = V; r.D = D; r.padding = padding_idx;
    r.wide = token_bytes == 8; r.table_dtype = weight_dtype; r.out_dtype = grad_dtype;
    r.scale = scale;
    r.workspace = workspace; r.workspace_bytes = workspace_bytes;
    r.stream = static_cast<hipStream_t>(stream);
    return ple::lookup_backward_run(r);
}

int ple_lookup_backward_plan_query(const void *grad_output, const void *grad_weight, int64_t T, int64_t V, int64_t D,
                                   int grad_dtype, int weight_dtype, ple_lookup_plan_info_t *info) {
    const int rc = ple::check_lookup(T, 1, V, D, false);
    if (rc != PLE_OK) return rc;
    if (!ple::valid_dtype(grad_dtype) || !ple::valid_dtype(weight_dtype)) return PLE_E_BAD_DTYPE;
    if (!info) return PLE_E_NULL_POINTER;
    ple::LookupRequest r{};
    r.grad = grad_output; r.dw = const_cast<void *>(grad_weight);
    r.T = T; r.F = 1; r.V = V; r.D = D;
    r.table_dtype = weight_dtype; r.out_dtype = grad_dtype;
    return ple::lookup_backward_plan_info(r, info);
}

int ple_residual_norm_launch(const void *residual, const void *branch, const ple_norm_t *norm, void *stream_out,
                             void *normed, float *stats, int64_t N, int64_t D, void *stream) {
    const int rc = ple::check_norm(norm, N, D);
    if (rc != PLE_OK) return rc;
    if (N == 0) return PLE_OK;
    // without a branch there is only the norm before the block
    if (!branch && (norm->post_norm != PLE_NORM_NONE || norm->gate || norm->residual_scale != 1.0f)) return PLE_E_UNSUPPORTED;
    if (!branch && norm->pre_norm == PLE_NORM_NONE) return PLE_E_UNSUPPORTED;
    if (!residual || !stats || (branch != nullptr) != (stream_out != nullptr) ||
        (norm->pre_norm != PLE_NORM_NONE) != (normed != nullptr))
        return PLE_E_NULL_POINTER;
    if (!ple::aligned_for(residual, norm->stream_dtype) || !ple::aligned_for(stream_out, norm->stream_dtype) ||
        !ple::aligned_for(branch, norm->branch_dtype) || !ple::aligned_for(normed, norm->branch_dtype) ||
        !ple::aligned(stats, 16))
        return PLE_E_MISALIGNED;
    ple::NormRequest r = ple::norm_request(norm, N, D, stream);
    r.residual = residual; r.branch = branch; r.stream_out = stream_out; r.normed = normed; r.stats = stats;
    return ple::norm_run(r);
}

size_t ple_residual_norm_backward_workspace_bytes(const ple_norm_t *norm, int64_t N, int64_t D) {
    if (ple::check_norm(norm, N, D) != PLE_OK) return 0;
    return ple::norm_backward_workspace_bytes(ple::norm_request(norm, N, D, nullptr));
}

int ple_residual_norm_backward_launch(const void *grad_stream, const void *grad_normed, const void *stream_in,
                                      const void *branch, const float *stats, const ple_norm_t *norm,
                                      const ple_norm_grads_t *grads, int64_t N, int64_t D, void *workspace,
                                      size_t workspace_bytes, void *stream) {
    const int rc = ple::check_norm(norm, N, D);
    if (rc != PLE_OK) return rc;
    if (!grads) return PLE_E_NULL_POINTER;
    // (an empty branch may have no address)
    if (N > 0 && !branch &&
        (norm->post_norm != PLE_NORM_NONE || norm->gate || norm->residual_scale != 1.0f || grads->branch))
        return PLE_E_UNSUPPORTED;
    if (grad_normed && norm->pre_norm == PLE_NORM_NONE) return PLE_E_UNSUPPORTED;
    if ((grads->post_weight && !norm->post_weight) || (grads->post_bias && !norm->post_bias) ||
        (grads->gate && !norm->gate) || (grads->pre_weight && !norm->pre_weight) || (grads->pre_bias && !norm->pre_bias))
        return PLE_E_NULL_POINTER;
    if (N > 0 && (!stats || (grad_normed && !stream_in))) return PLE_E_NULL_POINTER;
    for (const void *p : {grad_stream, stream_in, static_cast<const void *>(grads->residual)})
        if (!ple::aligned_for(p, norm->stream_dtype)) return PLE_E_MISALIGNED;
    for (const void *p : {grad_normed, branch, static_cast<const void *>(grads->branch)})
        if (!ple::aligned_for(p, norm->branch_dtype)) return PLE_E_MISALIGNED;
    for (const void *p : {grads->post_weight, grads->post_bias, grads->gate, grads->pre_weight, grads->pre_bias})
        if (!ple::aligned_for(p, norm->param_dtype)) return PLE_E_MISALIGNED;
    if (!ple::aligned(stats, 16)) return PLE_E_MISALIGNED;
    ple::NormRequest r = ple::norm_request(norm, N, D, stream);
    r.residual = stream_in; r.branch = branch; r.stats = const_cast<float *>(stats);
    r.g_stream = grad_stream; r.g_normed = grad_normed;
    r.d_residual = grads->residual; r.d_branch = grads->branch;
    r.d_post_w = grads->post_weight; r.d_post_b = grads->post_bias; r.d_gate = grads->gate;
    r.d_pre_w = grads->pre_weight; r.d_pre_b = grads->pre_bias;
    r.workspace = workspace; r.workspace_bytes = workspace_bytes;
    return ple::norm_backward_run(r);
}

size_t ple_distill_workspace_bytes(int64_t N, int64_t V) {
    if (N < 1 || V < 1 || V > (int64_t{1} << 30) || N > (int64_t{1} << 40) / V || N > (1 << 24)) return 0;
    return ple::distill_workspace_bytes(N, V);
}

int ple_distill_launch(const void *logits, const void *teacher_logits, const void *teacher_classes, int class_bytes,
                       const float *teacher_lse, const int64_t *labels, float *loss, float *stats, int64_t N, int64_t V,
                       int64_t K, float temperature, float alpha, int dtype, int teacher_dtype, void *workspace,
                       size_t workspace_bytes, void *stream) {
    const int rc = ple::check_distill(N, V, K, dtype, teacher_dtype, class_bytes, temperature, alpha);
    if (rc != PLE_OK) return rc;
    if (N == 0) return PLE_OK;
    if (!logits || !teacher_logits || !teacher_classes || !loss || !stats) return PLE_E_NULL_POINTER;
    if (!ple::aligned_for(logits, dtype) || !ple::aligned_for(teacher_logits, teacher_dtype) ||
        !ple::aligned(teacher_classes, class_bytes) || !ple::aligned(teacher_lse, 4) || !ple::aligned(labels, 8) ||
        !ple::aligned(loss, 4) || !ple::aligned(stats, 16))
        return PLE_E_MISALIGNED;
    ple::DistillRequest r{};
    r.logits = logits; r.teacher = teacher_logits; r.classes = teacher_classes;
    r.teacher_lse = teacher_lse; r.labels = labels; r.loss = loss; r.stats = stats;
    r.N = N; r.V = V; r.K = K;
    r.dtype = dtype; r.teacher_dtype = teacher_dtype; r.wide = class_bytes == 8;
    r.temperature = temperature; r.alpha = alpha;
    r.workspace = workspace; r.workspace_bytes = workspace_bytes;
    r.stream = static_cast<hipStream_t>(stream);
    return ple::distill_run(r);
}

int ple_distill_backward_launch(const float *grad_loss, const void *logits, const void *teacher_logits,
                                const void *teacher_classes, int class_bytes, const int64_t *labels, const float *stats,
                                void *grad_logits, int64_t N, int64_t V, int64_t K, float temperature, float alpha,
                                int dtype, int teacher_dtype, void *stream) {
    const int rc = ple::check_distill(N, V, K, dtype, teacher_dtype, class_bytes, temperature, alpha);
    if (rc != PLE_OK) return rc;
    if (N == 0) return PLE_OK;
    if (!grad_loss || !logits || !teacher_logits || !teacher_classes || !stats || !grad_logits) return PLE_E_NULL_POINTER;
    if (!ple::aligned_for(logits, dtype) || !ple::aligned_for(grad_logits, dtype) ||
        !ple::aligned_for(teacher_logits, teacher_dtype) || !ple::aligned(teacher_classes, class_bytes) ||
        !ple::aligned(labels, 8) || !ple::aligned(grad_loss, 4) || !ple::aligned(stats, 16))
        return PLE_E_MISALIGNED;
    ple::DistillRequest r{};
    r.logits = logits; r.teacher = teacher_logits; r.classes = teacher_classes; r.labels = labels;
    r.g = grad_loss; r.dz = grad_logits; r.stats = const_cast<float *>(stats);
    r.N = N; r.V = V; r.K = K;
    r.dtype = dtype; r.teacher_dtype = teacher_dtype; r.wide = class_bytes == 8;
    r.temperature = temperature; r.alpha = alpha;
    r.stream = static_cast<hipStream_t>(stream);
    return ple::distill_backward_run(r);
}

}  // extern "C"

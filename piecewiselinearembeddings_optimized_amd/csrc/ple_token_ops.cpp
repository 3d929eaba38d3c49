// PyTorch dispatcher registration of the operators around the embedding:
// lookup (tokens and categorical columns), residual_norm (the norms after and
// before a block with its gate and residual scale) and distillation_loss, each
// with its backward.  Host code only, as ple_ops.cpp: it validates the tensors,
// allocates outputs and scratch with the ATen caching allocator, and calls the
// C ABI of include/ple_hip.h on the caller's current HIP stream, without a host
// synchronisation.

#include <torch/library.h>

#include <array>
#include <limits>
#include <tuple>

#include "ple_torch.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

bool is_float_type(at::ScalarType t) { return ple_dtype_of(t) >= 0; }

bool is_index_type(at::ScalarType t) { return t == at::kInt || t == at::kLong; }

void check_tensor(const Tensor &t, const Tensor &like, const char *name) {
    TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on the same CUDA device as the other tensors");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

const void *opt_ptr(const OptTensor &t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }

bool has(const OptTensor &t) { return t.has_value() && t->defined(); }

Tensor scratch(size_t bytes, const Tensor &like) {
    return at::empty({static_cast<int64_t>(bytes > 0 ? bytes : 1)}, like.options().dtype(at::kByte));
}

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------

int64_t check_tokens(const Tensor &tokens, const OptTensor &offsets, const Tensor &like) {
    check_tensor(tokens, like, "tokens");
    TORCH_CHECK(is_index_type(tokens.scalar_type()), "tokens must be int32 or int64");
    if (!has(offsets)) return 1;
    check_tensor(*offsets, like, "offsets");
    TORCH_CHECK(offsets->scalar_type() == at::kLong && offsets->dim() == 1 && offsets->size(0) >= 2,
                "offsets must be int64 [F + 1]");
    const int64_t F = offsets->size(0) - 1;
    TORCH_CHECK(tokens.dim() >= 1 && tokens.size(-1) == F, "the last dimension of tokens must be offsets.size(0) - 1");
    return F;
}

at::DimVector with_width(const Tensor &tokens, int64_t D) {
    at::DimVector shape(tokens.sizes().begin(), tokens.sizes().end());
    shape.push_back(D);
    return shape;
}

Tensor ple_lookup(const Tensor &tokens, const Tensor &weight, const OptTensor &offsets, double scale, int64_t padding_idx,
                  at::ScalarType output_dtype) {
    TORCH_CHECK(weight.is_cuda(), "weight must be a CUDA tensor");
    check_tensor(weight, weight, "weight");
    const int64_t F = check_tokens(tokens, offsets, weight);
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0, "weight must have shape [V, D]");
    TORCH_CHECK(is_float_type(weight.scalar_type()), "weight must be float32, float16, or bfloat16");
    TORCH_CHECK(is_float_type(output_dtype), "output_dtype must be float32, float16, or bfloat16");
    const int64_t V = weight.size(0), D = weight.size(1), T = tokens.numel();
    DeviceScope scope(weight.device().index());
    Tensor out = at::empty(with_width(tokens, D), weight.options().dtype(output_dtype));
    if (T == 0) return out;
    const int rc = ple_lookup_launch(tokens.data_ptr(), static_cast<int>(tokens.element_size()),
                                     static_cast<const int64_t *>(opt_ptr(offsets)), weight.data_ptr(), out.data_ptr(), T,
                                     F, V, D, static_cast<float>(scale), ple_dtype_of(weight.scalar_type()),
                                     ple_dtype_of(output_dtype), current_stream(weight));
    check_rc(rc, "ple_lookup_launch");
    return out;
}

Tensor ple_lookup_backward(const Tensor &grad_output, const Tensor &tokens, const OptTensor &offsets, int64_t num_rows,
                           double scale, int64_t padding_idx, at::ScalarType grad_dtype) {
    TORCH_CHECK(grad_output.is_cuda(), "grad_output must be a CUDA tensor");
    check_tensor(grad_output, grad_output, "grad_output");
    const int64_t F = check_tokens(tokens, offsets, grad_output);
    TORCH_CHECK(grad_output.dim() == tokens.dim() + 1 && grad_output.sizes().slice(0, tokens.dim()) == tokens.sizes() &&
                    grad_output.size(-1) > 0,
                "grad_output must have the shape of tokens and one more dimension");
    TORCH_CHECK(is_float_type(grad_output.scalar_type()), "grad_output must be float32, float16, or bfloat16");
    TORCH_CHECK(is_float_type(grad_dtype), "grad_dtype must be float32, float16, or bfloat16");
    TORCH_CHECK(num_rows > 0, "num_rows must be positive");
    const int64_t D = grad_output.size(-1), T = tokens.numel();
    DeviceScope scope(grad_output.device().index());
    Tensor grad_weight = at::empty({num_rows, D}, grad_output.options().dtype(grad_dtype));
    const size_t bytes = ple_lookup_backward_workspace_bytes(T, num_rows, D);
    Tensor ws = scratch(bytes, grad_output);
    const int rc = ple_lookup_backward_launch(
        grad_output.data_ptr(), tokens.data_ptr(), static_cast<int>(tokens.element_size()),
        static_cast<const int64_t *>(opt_ptr(offsets)), grad_weight.data_ptr(), T, F, num_rows, D, padding_idx,
        static_cast<float>(scale), ple_dtype_of(grad_output.scalar_type()), ple_dtype_of(grad_dtype), ws.data_ptr(), bytes,
        current_stream(grad_output));
    check_rc(rc, "ple_lookup_backward_launch");
    return grad_weight;
}

// ---------------------------------------------------------------------------
// residual_norm
// ---------------------------------------------------------------------------

// The descriptor of a call; `stream` and `branch_type` give the types.
ple_norm_t describe_norm(const Tensor &stream, at::ScalarType branch_type, const OptTensor &post_weight,
                         const OptTensor &post_bias, const OptTensor &gate, const OptTensor &pre_weight,
                         const OptTensor &pre_bias, int64_t post_norm, int64_t pre_norm, int64_t gate_activation,
                         double residual_scale, double eps) {
    TORCH_CHECK(stream.dim() >= 1 && stream.size(-1) > 0, "the residual stream must have shape [..., D]");
    TORCH_CHECK(is_float_type(stream.scalar_type()), "the residual stream must be float32, float16, or bfloat16");
    TORCH_CHECK(is_float_type(branch_type), "the branch must be float32, float16, or bfloat16");
    TORCH_CHECK(stream.scalar_type() == at::kFloat || stream.scalar_type() == branch_type,
                "the residual stream must be float32 or of the branch's dtype");
    TORCH_CHECK(post_norm >= 0 && post_norm <= 2 && pre_norm >= 0 && pre_norm <= 2,
                "post_norm and pre_norm must be 0 (none), 1 (rms) or 2 (layer)");
    TORCH_CHECK(gate_activation >= 0 && gate_activation <= 2, "gate_activation must be 0 (none), 1 (sigmoid) or 2 (tanh)");
    TORCH_CHECK(post_norm != 0 || (!has(post_weight) && !has(post_bias)), "post_weight and post_bias need a post norm");
    TORCH_CHECK(pre_norm != 0 || (!has(pre_weight) && !has(pre_bias)), "pre_weight and pre_bias need a pre norm");
    const int64_t D = stream.size(-1), N = stream.numel() / D;
    TORCH_CHECK(D <= PLE_NORM_MAX_WIDTH, "rows of at most ", PLE_NORM_MAX_WIDTH, " elements are supported, got ", D);
    ple_norm_t d{};
    d.param_dtype = PLE_DTYPE_F32;
    at::ScalarType param_type = at::ScalarType::Undefined;
    const auto param = [&](const OptTensor &t, const char *name, bool rows) -> const void * {
        if (!has(t)) return nullptr;
        check_tensor(*t, stream, name);
        TORCH_CHECK(is_float_type(t->scalar_type()), name, " must be float32, float16, or bfloat16");
        TORCH_CHECK(param_type == at::ScalarType::Undefined || param_type == t->scalar_type(),
                    "weights, biases and the gate must have one dtype");
        param_type = t->scalar_type();
        if (rows) {
            TORCH_CHECK(t->dim() == 2 && t->size(1) == D, name, " must have shape [G, D]");
        } else {
            TORCH_CHECK(t->dim() == 1 && t->size(0) == D, name, " must have shape [D]");
        }
        return t->data_ptr();
    };
    d.post_weight = param(post_weight, "post_weight", false);
    d.post_bias = param(post_bias, "post_bias", false);
    d.gate = param(gate, "gate", true);
    d.pre_weight = param(pre_weight, "pre_weight", false);
    d.pre_bias = param(pre_bias, "pre_bias", false);
    if (d.gate) {
        d.gate_rows = gate->size(0);
        TORCH_CHECK(d.gate_rows > 0 && (N == 0 || (d.gate_rows <= N && N % d.gate_rows == 0)),
                    "the gate's rows must divide the number of rows");
    }
    if (param_type != at::ScalarType::Undefined) d.param_dtype = ple_dtype_of(param_type);
    d.post_norm = static_cast<int>(post_norm);
    d.pre_norm = static_cast<int>(pre_norm);
    d.gate_activation = static_cast<int>(gate_activation);
    d.stream_dtype = ple_dtype_of(stream.scalar_type());
    d.branch_dtype = ple_dtype_of(branch_type);
    d.residual_scale = static_cast<float>(residual_scale);
    d.eps = static_cast<float>(eps);
    return d;
}

void check_branch(const OptTensor &branch, const Tensor &stream, int64_t post_norm, const OptTensor &gate,
                  double residual_scale) {
    if (has(branch)) {
        check_tensor(*branch, stream, "branch");
        TORCH_CHECK(branch->sizes() == stream.sizes(), "branch must have the shape of the residual stream");
    } else {
        TORCH_CHECK(post_norm == 0 && !has(gate) && residual_scale == 1.0,
                    "without a branch there is no post norm, no gate and no residual scale");
    }
}

std::tuple<Tensor, Tensor, Tensor> ple_residual_norm(
    const Tensor &residual, const OptTensor &branch, const OptTensor &post_weight, const OptTensor &post_bias,
    const OptTensor &gate, const OptTensor &pre_weight, const OptTensor &pre_bias, int64_t post_norm, int64_t pre_norm,
    int64_t gate_activation, double residual_scale, double eps, at::ScalarType normed_dtype) {
    TORCH_CHECK(residual.is_cuda(), "residual must be a CUDA tensor");
    check_tensor(residual, residual, "residual");
    check_branch(branch, residual, post_norm, gate, residual_scale);
    TORCH_CHECK(!has(branch) || branch->scalar_type() == normed_dtype, "normed_dtype must be the branch's dtype");
    TORCH_CHECK(has(branch) || pre_norm != 0, "without a branch there has to be a pre norm");
    const ple_norm_t d = describe_norm(residual, normed_dtype, post_weight, post_bias, gate, pre_weight, pre_bias, post_norm,
                                       pre_norm, gate_activation, residual_scale, eps);
    const int64_t D = residual.size(-1), N = residual.numel() / D;
    DeviceScope scope(residual.device().index());
    Tensor stream = has(branch) ? at::empty_like(residual) : at::empty({0}, residual.options());
    Tensor normed = pre_norm != 0 ? at::empty_like(residual, residual.options().dtype(normed_dtype))
                                  : at::empty({0}, residual.options().dtype(normed_dtype));
    Tensor stats = at::empty({N, 4}, residual.options().dtype(at::kFloat));
    if (N == 0) return {stream, normed, stats};
    const int rc = ple_residual_norm_launch(residual.data_ptr(), opt_ptr(branch), &d,
                                            has(branch) ? stream.data_ptr() : nullptr,
                                            pre_norm != 0 ? normed.data_ptr() : nullptr, stats.data_ptr<float>(), N, D,
                                            current_stream(residual));
    check_rc(rc, "ple_residual_norm_launch");
    return {stream, normed, stats};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> ple_residual_norm_backward(
    const OptTensor &grad_stream, const OptTensor &grad_normed, const Tensor &stream, const OptTensor &branch,
    const Tensor &stats, const OptTensor &post_weight, const OptTensor &post_bias, const OptTensor &gate,
    const OptTensor &pre_weight, const OptTensor &pre_bias, int64_t post_norm, int64_t pre_norm, int64_t gate_activation,
    double residual_scale, std::array<bool, 7> output_mask) {
    TORCH_CHECK(stream.is_cuda(), "stream must be a CUDA tensor");
    check_tensor(stream, stream, "stream");
    check_branch(branch, stream, post_norm, gate, residual_scale);
    const at::ScalarType branch_type = has(branch) ? branch->scalar_type()
                                                   : (has(grad_normed) ? grad_normed->scalar_type() : stream.scalar_type());
    const ple_norm_t d = describe_norm(stream, branch_type, post_weight, post_bias, gate, pre_weight, pre_bias, post_norm,
                                       pre_norm, gate_activation, residual_scale, 0.0);
    const int64_t D = stream.size(-1), N = stream.numel() / D;
    check_tensor(stats, stream, "stats");
    TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.dim() == 2 && stats.size(0) == N && stats.size(1) == 4,
                "stats must be the float32 [N, 4] of the forward");
    if (has(grad_stream)) {
        check_tensor(*grad_stream, stream, "grad_stream");
        TORCH_CHECK(grad_stream->sizes() == stream.sizes() && grad_stream->scalar_type() == stream.scalar_type(),
                    "grad_stream must have the shape and dtype of stream");
    }
    if (has(grad_normed)) {
        TORCH_CHECK(pre_norm != 0, "grad_normed needs a pre norm");
        check_tensor(*grad_normed, stream, "grad_normed");
        TORCH_CHECK(grad_normed->sizes() == stream.sizes() && grad_normed->scalar_type() == branch_type,
                    "grad_normed must have the shape of stream and the branch's dtype");
    }
    DeviceScope scope(stream.device().index());
    ple_norm_grads_t g{};
    const auto out = [&](bool wanted, const OptTensor &like, void *&p) {
        if (!wanted || !has(like)) return at::empty({0}, stream.options());
        Tensor t = at::empty_like(*like);
        p = t.data_ptr();
        return t;
    };
    Tensor d_residual = out(output_mask[0], stream, g.residual);
    Tensor d_branch = out(output_mask[1], branch, g.branch);
    Tensor d_post_weight = out(output_mask[2], post_weight, g.post_weight);
    Tensor d_post_bias = out(output_mask[3], post_bias, g.post_bias);
    Tensor d_gate = out(output_mask[4], gate, g.gate);
    Tensor d_pre_weight = out(output_mask[5], pre_weight, g.pre_weight);
    Tensor d_pre_bias = out(output_mask[6], pre_bias, g.pre_bias);
    const size_t bytes = ple_residual_norm_backward_workspace_bytes(&d, N, D);
    Tensor ws = scratch(bytes, stream);
    const int rc = ple_residual_norm_backward_launch(opt_ptr(grad_stream), opt_ptr(grad_normed), stream.data_ptr(),
                                                     opt_ptr(branch), stats.data_ptr<float>(), &d, &g, N, D, ws.data_ptr(),
                                                     bytes, current_stream(stream));
    check_rc(rc, "ple_residual_norm_backward_launch");
    return {d_residual, d_branch, d_post_weight, d_post_bias, d_gate, d_pre_weight, d_pre_bias};
}

// ---------------------------------------------------------------------------
// distillation_loss
// ---------------------------------------------------------------------------

void check_distillation(const Tensor &logits, const Tensor &teacher_logits, const Tensor &teacher_classes,
                        const OptTensor &labels, double temperature, double alpha) {
    TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
    check_tensor(logits, logits, "logits");
    check_tensor(teacher_logits, logits, "teacher_logits");
    check_tensor(teacher_classes, logits, "teacher_classes");
    TORCH_CHECK(logits.dim() == 2 && logits.size(1) > 0, "logits must have shape [N, V]");
    TORCH_CHECK(is_float_type(logits.scalar_type()), "logits must be float32, float16, or bfloat16");
    TORCH_CHECK(teacher_logits.dim() == 2 && teacher_logits.size(0) == logits.size(0) && teacher_logits.size(1) > 0,
                "teacher_logits must have shape [N, K]");
    TORCH_CHECK(is_float_type(teacher_logits.scalar_type()), "teacher_logits must be float32, float16, or bfloat16");
    TORCH_CHECK(teacher_classes.sizes() == teacher_logits.sizes(), "teacher_classes must have shape [N, K]");
    TORCH_CHECK(is_index_type(teacher_classes.scalar_type()), "teacher_classes must be int32 or int64");
    if (has(labels)) {
        check_tensor(*labels, logits, "labels");
        TORCH_CHECK(labels->scalar_type() == at::kLong && labels->dim() == 1 && labels->size(0) == logits.size(0),
                    "labels must be int64 [N]");
    }
    TORCH_CHECK(temperature > 1e-6 && temperature < 1e6, "temperature must be between 1e-6 and 1e6, got ", temperature);
    TORCH_CHECK(alpha >= 0.0 && alpha <= 1.0, "alpha must be between 0 and 1, got ", alpha);
}

std::tuple<Tensor, Tensor> ple_distillation_loss(const Tensor &logits, const Tensor &teacher_logits,
                                                 const Tensor &teacher_classes, const OptTensor &teacher_lse,
                                                 const OptTensor &labels, double temperature, double alpha) {
    check_distillation(logits, teacher_logits, teacher_classes, labels, temperature, alpha);
    const int64_t N = logits.size(0), V = logits.size(1), K = teacher_logits.size(1);
    if (has(teacher_lse)) {
        check_tensor(*teacher_lse, logits, "teacher_lse");
        TORCH_CHECK(teacher_lse->scalar_type() == at::kFloat && teacher_lse->dim() == 1 && teacher_lse->size(0) == N,
                    "teacher_lse must be float32 [N]");
    }
    DeviceScope scope(logits.device().index());
    Tensor loss = at::empty({N}, logits.options().dtype(at::kFloat));
    Tensor stats = at::empty({N, PLE_DISTILL_STATS}, logits.options().dtype(at::kFloat));
    if (N == 0) return {loss, stats};
    const size_t bytes = ple_distill_workspace_bytes(N, V);
    Tensor ws;
    if (bytes > 0) ws = scratch(bytes, logits);
    const int rc = ple_distill_launch(
        logits.data_ptr(), teacher_logits.data_ptr(), teacher_classes.data_ptr(),
        static_cast<int>(teacher_classes.element_size()), static_cast<const float *>(opt_ptr(teacher_lse)),
        static_cast<const int64_t *>(opt_ptr(labels)), loss.data_ptr<float>(), stats.data_ptr<float>(), N, V, K,
        static_cast<float>(temperature), static_cast<float>(alpha), ple_dtype_of(logits.scalar_type()),
        ple_dtype_of(teacher_logits.scalar_type()), bytes > 0 ? ws.data_ptr() : nullptr, bytes, current_stream(logits));
    check_rc(rc, "ple_distill_launch");
    return {loss, stats};
}

Tensor ple_distillation_loss_backward(const Tensor &grad_loss, const Tensor &logits, const Tensor &teacher_logits,
                                      const Tensor &teacher_classes, const OptTensor &labels, const Tensor &stats,
                                      double temperature, double alpha) {
    check_distillation(logits, teacher_logits, teacher_classes, labels, temperature, alpha);
    const int64_t N = logits.size(0), V = logits.size(1), K = teacher_logits.size(1);
    check_tensor(grad_loss, logits, "grad_loss");
    TORCH_CHECK(grad_loss.scalar_type() == at::kFloat && grad_loss.dim() == 1 && grad_loss.size(0) == N,
                "grad_loss must be float32 [N]");
    check_tensor(stats, logits, "stats");
    TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.dim() == 2 && stats.size(0) == N &&
                    stats.size(1) == PLE_DISTILL_STATS,
                "stats must be the float32 statistics of the forward");
    DeviceScope scope(logits.device().index());
    Tensor grad_logits = at::empty_like(logits);
    if (N == 0) return grad_logits;
    const int rc = ple_distill_backward_launch(
        grad_loss.data_ptr<float>(), logits.data_ptr(), teacher_logits.data_ptr(), teacher_classes.data_ptr(),
        static_cast<int>(teacher_classes.element_size()), static_cast<const int64_t *>(opt_ptr(labels)),
        stats.data_ptr<float>(), grad_logits.data_ptr(), N, V, K, static_cast<float>(temperature),
        static_cast<float>(alpha), ple_dtype_of(logits.scalar_type()), ple_dtype_of(teacher_logits.scalar_type()),
        current_stream(logits));
    check_rc(rc, "ple_distill_backward_launch");
    return grad_logits;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(rtdl_num_embeddings_cuda, m) {
    m.def(
        "lookup(Tensor tokens, Tensor weight, Tensor? offsets, float scale, int padding_idx, ScalarType output_dtype) "
        "-> Tensor");
    m.def(
        "lookup_backward(Tensor grad_output, Tensor tokens, Tensor? offsets, int num_rows, float scale, "
        "int padding_idx, ScalarType grad_dtype) -> Tensor");
    m.def(
        "residual_norm(Tensor residual, Tensor? branch, Tensor? post_weight, Tensor? post_bias, Tensor? gate, "
        "Tensor? pre_weight, Tensor? pre_bias, int post_norm, int pre_norm, int gate_activation, float residual_scale, "
        "float eps, ScalarType normed_dtype) -> (Tensor stream, Tensor normed, Tensor stats)");
    m.def(
        "residual_norm_backward(Tensor? grad_stream, Tensor? grad_normed, Tensor stream, Tensor? branch, Tensor stats, "
        "Tensor? post_weight, Tensor? post_bias, Tensor? gate, Tensor? pre_weight, Tensor? pre_bias, int post_norm, "
        "int pre_norm, int gate_activation, float residual_scale, bool[7] output_mask) -> (Tensor grad_residual, "
        "Tensor grad_branch, Tensor grad_post_weight, Tensor grad_post_bias, Tensor grad_gate, Tensor grad_pre_weight, "
        "Tensor grad_pre_bias)");
    m.def(
        "distillation_loss(Tensor logits, Tensor teacher_logits, Tensor teacher_classes, Tensor? teacher_lse, "
        "Tensor? labels, float temperature, float alpha) -> (Tensor loss, Tensor stats)");
    m.def(
        "distillation_loss_backward(Tensor grad_loss, Tensor logits, Tensor teacher_logits, Tensor teacher_classes, "
        "Tensor? labels, Tensor stats, float temperature, float alpha) -> Tensor grad_logits");
}

TORCH_LIBRARY_IMPL(rtdl_num_embeddings_cuda, CUDA, m) {
    m.impl("lookup", &ple_lookup);
    m.impl("lookup_backward", &ple_lookup_backward);
    m.impl("residual_norm", &ple_residual_norm);
    m.impl("residual_norm_backward", &ple_residual_norm_backward);
    m.impl("distillation_loss", &ple_distillation_loss);
    m.impl("distillation_loss_backward", &ple_distillation_loss_backward);
}

// Autograd formulas of the operators around the embedding, in C++ as
// ple_autograd.cpp's (and for the same reason).
//
// `lookup`: the gradient of `weight` from `lookup_backward`.
//
// `residual_norm`: gradients of the residual, the branch, the gate and the
// norms' parameters from one `residual_norm_backward`, which reads the stored
// stream (an output of the forward; the residual itself where there is no
// branch), the branch and the rows' statistics.  An output without a gradient
// is a zero gradient that is not read.  Statistics (the loss's too), and the empty
// output of a call that does not make it, are returned detached (compiled autograd
// refuses functions that mark outputs as not differentiable).
//
// `distillation_loss`: the gradient of the student's logits; the teacher is
// not learned, and a teacher that requires a gradient gets none.

#include <array>
#include <tuple>

#include "ple_autograd.h"

namespace {

using Tensors2 = std::tuple<Tensor, Tensor>;
using Tensors3 = std::tuple<Tensor, Tensor, Tensor>;
using Tensors7 = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;

PLE_OP(op_lookup, "lookup", Tensor(const Tensor &, const Tensor &, const OptTensor &, double, int64_t, at::ScalarType))
PLE_OP(op_lookup_backward, "lookup_backward",
       Tensor(const Tensor &, const Tensor &, const OptTensor &, int64_t, double, int64_t, at::ScalarType))
PLE_OP(op_residual_norm, "residual_norm",
       Tensors3(const Tensor &, const OptTensor &, const OptTensor &, const OptTensor &, const OptTensor &,
                const OptTensor &, const OptTensor &, int64_t, int64_t, int64_t, double, double, at::ScalarType))
PLE_OP(op_residual_norm_backward, "residual_norm_backward",
       Tensors7(const OptTensor &, const OptTensor &, const Tensor &, const OptTensor &, const Tensor &,
                const OptTensor &, const OptTensor &, const OptTensor &, const OptTensor &, const OptTensor &, int64_t,
                int64_t, int64_t, double, std::array<bool, 7>))
PLE_OP(op_distillation_loss, "distillation_loss",
       Tensors2(const Tensor &, const Tensor &, const Tensor &, const OptTensor &, const OptTensor &, double, double))
PLE_OP(op_distillation_loss_backward, "distillation_loss_backward",
       Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &, const OptTensor &, const Tensor &, double,
              double))

OptTensor maybe(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }

OptTensor maybe_contiguous(const Tensor &t) { return t.defined() ? OptTensor(t.contiguous()) : OptTensor(); }

struct Lookup : torch::autograd::Function<Lookup> {
    static constexpr bool is_traceable = true;
    static Tensor forward(AutogradContext *ctx, DispatchKeySet ks, const Tensor &tokens, const Tensor &weight,
                          const OptTensor &offsets, double scale, int64_t padding_idx, at::ScalarType output_dtype) {
        at::AutoDispatchBelowAutograd guard;
        Tensor out = op_lookup().redispatch(below(ks), tokens, weight, offsets, scale, padding_idx, output_dtype);
        ctx->save_for_backward({tokens, offsets.value_or(Tensor())});
        ctx->saved_data["rows"] = weight.size(0);
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding"] = padding_idx;
        ctx->saved_data["dtype"] = static_cast<int64_t>(weight.scalar_type());
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list r(7);
        if (!grads[0].defined()) return r;
        const auto s = ctx->get_saved_variables();
        r[2] = op_lookup_backward().call(grads[0].contiguous(), s[0], maybe(s[1]), ctx->saved_data["rows"].toInt(),
                                         ctx->saved_data["scale"].toDouble(), ctx->saved_data["padding"].toInt(),
                                         static_cast<at::ScalarType>(ctx->saved_data["dtype"].toInt()));
        return r;
    }
};

Tensor lookup(DispatchKeySet ks, const Tensor &tokens, const Tensor &weight, const OptTensor &offsets, double scale,
              int64_t padding_idx, at::ScalarType output_dtype) {
    if (!recorded(weight)) {
        at::AutoDispatchBelowAutograd guard;
        return op_lookup().redispatch(below(ks), tokens, weight, offsets, scale, padding_idx, output_dtype);
    }
    return Lookup::apply(ks, tokens, weight, offsets, scale, padding_idx, output_dtype);
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static constexpr bool is_traceable = true;
    static variable_list forward(AutogradContext *ctx, DispatchKeySet ks, const Tensor &residual, const OptTensor &branch,
                                 const OptTensor &post_weight, const OptTensor &post_bias, const OptTensor &gate,
                                 const OptTensor &pre_weight, const OptTensor &pre_bias, int64_t post_norm,
                                 int64_t pre_norm, int64_t gate_activation, double residual_scale, double eps,
                                 at::ScalarType normed_dtype) {
        at::AutoDispatchBelowAutograd guard;
        auto [stream, normed, stats] =
            op_residual_norm().redispatch(below(ks), residual, branch, post_weight, post_bias, gate, pre_weight, pre_bias,
                                          post_norm, pre_norm, gate_activation, residual_scale, eps, normed_dtype);
        const bool has_branch = branch.has_value() && branch->defined();
        ctx->save_for_backward({has_branch ? stream : residual, branch.value_or(Tensor()), stats,
                                post_weight.value_or(Tensor()), post_bias.value_or(Tensor()), gate.value_or(Tensor()),
                                pre_weight.value_or(Tensor()), pre_bias.value_or(Tensor())});
        ctx->saved_data["need"] = need_bits(residual, branch, post_weight, post_bias, gate, pre_weight, pre_bias);
        ctx->saved_data["post_norm"] = post_norm;
        ctx->saved_data["pre_norm"] = pre_norm;
        ctx->saved_data["gate_activation"] = gate_activation;
        ctx->saved_data["residual_scale"] = residual_scale;
        ctx->set_materialize_grads(false);
        return {stream, normed, stats};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list r(14);
        const auto s = ctx->get_saved_variables();
        const int64_t pre_norm = ctx->saved_data["pre_norm"].toInt();
        const bool has_branch = s[1].defined();
        // (an output that the call does not make has no gradient to pass on)
        const Tensor g_stream = has_branch ? grads[0] : Tensor();
        const Tensor g_normed = pre_norm != 0 ? grads[1] : Tensor();
        if (!g_stream.defined() && !g_normed.defined()) return r;
        const int64_t need = ctx->saved_data["need"].toInt();
        std::array<bool, 7> mask;
        for (int i = 0; i < 7; ++i) mask[i] = (need >> i) & 1;
        const Tensors7 g = op_residual_norm_backward().call(
            maybe_contiguous(g_stream), maybe_contiguous(g_normed), s[0], maybe(s[1]), s[2], maybe(s[3]), maybe(s[4]),
            maybe(s[5]), maybe(s[6]), maybe(s[7]), ctx->saved_data["post_norm"].toInt(), pre_norm,
            ctx->saved_data["gate_activation"].toInt(), ctx->saved_data["residual_scale"].toDouble(), mask);
        r[1] = if_bit(need, 0, std::get<0>(g));
        r[2] = if_bit(need, 1, std::get<1>(g));
        r[3] = if_bit(need, 2, std::get<2>(g));
        r[4] = if_bit(need, 3, std::get<3>(g));
        r[5] = if_bit(need, 4, std::get<4>(g));
        r[6] = if_bit(need, 5, std::get<5>(g));
        r[7] = if_bit(need, 6, std::get<6>(g));
        return r;
    }
};

Tensors3 residual_norm(DispatchKeySet ks, const Tensor &residual, const OptTensor &branch, const OptTensor &post_weight,
                       const OptTensor &post_bias, const OptTensor &gate, const OptTensor &pre_weight,
                       const OptTensor &pre_bias, int64_t post_norm, int64_t pre_norm, int64_t gate_activation,
                       double residual_scale, double eps, at::ScalarType normed_dtype) {
    if (!recorded(residual, branch, post_weight, post_bias, gate, pre_weight, pre_bias)) {
        at::AutoDispatchBelowAutograd guard;
        return op_residual_norm().redispatch(below(ks), residual, branch, post_weight, post_bias, gate, pre_weight,
                                             pre_bias, post_norm, pre_norm, gate_activation, residual_scale, eps,
                                             normed_dtype);
    }
    auto r = ResidualNorm::apply(ks, residual, branch, post_weight, post_bias, gate, pre_weight, pre_bias, post_norm,
                                 pre_norm, gate_activation, residual_scale, eps, normed_dtype);
    const bool has_branch = branch.has_value() && branch->defined();
    return {has_branch ? r[0] : r[0].detach(), pre_norm != 0 ? r[1] : r[1].detach(), r[2].detach()};
}

struct DistillationLoss : torch::autograd::Function<DistillationLoss> {
    static constexpr bool is_traceable = true;
    static variable_list forward(AutogradContext *ctx, DispatchKeySet ks, const Tensor &logits,
                                 const Tensor &teacher_logits, const Tensor &teacher_classes,
                                 const OptTensor &teacher_lse, const OptTensor &labels, double temperature, double alpha) {
        at::AutoDispatchBelowAutograd guard;
        auto [loss, stats] = op_distillation_loss().redispatch(below(ks), logits, teacher_logits, teacher_classes,
                                                               teacher_lse, labels, temperature, alpha);
        ctx->save_for_backward({logits, teacher_logits, teacher_classes, labels.value_or(Tensor()), stats});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["alpha"] = alpha;
        ctx->set_materialize_grads(false);
        return {loss, stats};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list r(8);
        if (!grads[0].defined()) return r;
        const auto s = ctx->get_saved_variables();
        r[1] = op_distillation_loss_backward().call(grads[0].contiguous(), s[0], s[1], s[2], maybe(s[3]), s[4],
                                                    ctx->saved_data["temperature"].toDouble(),
                                                    ctx->saved_data["alpha"].toDouble());
        return r;
    }
};

Tensors2 distillation_loss(DispatchKeySet ks, const Tensor &logits, const Tensor &teacher_logits,
                           const Tensor &teacher_classes, const OptTensor &teacher_lse, const OptTensor &labels,
                           double temperature, double alpha) {
    if (!recorded(logits)) {
        at::AutoDispatchBelowAutograd guard;
        return op_distillation_loss().redispatch(below(ks), logits, teacher_logits, teacher_classes, teacher_lse, labels,
                                                 temperature, alpha);
    }
    auto r = DistillationLoss::apply(ks, logits, teacher_logits, teacher_classes, teacher_lse, labels, temperature, alpha);
    return {r[0], r[1].detach()};
}

}  // namespace

TORCH_LIBRARY_IMPL(rtdl_num_embeddings_cuda, Autograd, m) {
    m.impl("lookup", TORCH_FN(lookup));
    m.impl("residual_norm", TORCH_FN(residual_norm));
    m.impl("distillation_loss", TORCH_FN(distillation_loss));
}

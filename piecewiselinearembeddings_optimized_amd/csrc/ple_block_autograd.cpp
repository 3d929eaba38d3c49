// Autograd formulas of group_norm and relative_bias, in C++ as ple_autograd.cpp's
// (and for the same reason).  The group norm's backward reads its input and the
// forward's statistics, which are returned detached; the relative bias's only its
// buckets.  The gradients' norm and clipping are not differentiable.

#include <array>
#include <tuple>

#include "ple_autograd.h"

namespace {

using c10::SymInt;
using Tensors2 = std::tuple<Tensor, Tensor>;
using Tensors3 = std::tuple<Tensor, Tensor, Tensor>;

PLE_OP(op_group_norm, "group_norm", Tensors2(const Tensor &, const OptTensor &, const OptTensor &, int64_t, int64_t, double))
PLE_OP(op_group_norm_backward, "group_norm_backward",
       Tensors3(const Tensor &, const Tensor &, const Tensor &, const OptTensor &, const OptTensor &, int64_t, int64_t,
                std::array<bool, 3>))
PLE_OP(op_relative_bias, "relative_bias",
       Tensor(const Tensor &, const Tensor &, const OptTensor &, SymInt, SymInt, SymInt, bool, at::ScalarType))
PLE_OP(op_relative_bias_backward, "relative_bias_backward",
       Tensor(const Tensor &, const Tensor &, const OptTensor &, SymInt, SymInt, bool, at::ScalarType))

OptTensor maybe(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct GroupNorm : torch::autograd::Function<GroupNorm> {
    static constexpr bool is_traceable = true;
    static variable_list forward(AutogradContext *ctx, DispatchKeySet ks, const Tensor &x, const OptTensor &weight,
                                 const OptTensor &bias, int64_t num_groups, int64_t activation, double eps) {
        at::AutoDispatchBelowAutograd guard;
        auto [y, stats] = op_group_norm().redispatch(below(ks), x, weight, bias, num_groups, activation, eps);
        ctx->save_for_backward({x, stats, weight.value_or(Tensor()), bias.value_or(Tensor())});
        ctx->saved_data["need"] = need_bits(x, weight, bias);
        ctx->saved_data["groups"] = num_groups;
        ctx->saved_data["activation"] = activation;
        ctx->set_materialize_grads(false);
        return {y, stats};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list r(7);
        if (!grads[0].defined()) return r;
        const auto s = ctx->get_saved_variables();
        const int64_t need = ctx->saved_data["need"].toInt();
        const std::array<bool, 3> mask{(need & 1) != 0, (need & 2) != 0, (need & 4) != 0};
        const Tensors3 g = op_group_norm_backward().call(grads[0].contiguous(), s[0], s[1], maybe(s[2]), maybe(s[3]),
                                                         ctx->saved_data["groups"].toInt(),
                                                         ctx->saved_data["activation"].toInt(), mask);
        r[1] = if_bit(need, 0, std::get<0>(g));
        r[2] = if_bit(need, 1, std::get<1>(g));
        r[3] = if_bit(need, 2, std::get<2>(g));
        return r;
    }
};

Tensors2 group_norm(DispatchKeySet ks, const Tensor &x, const OptTensor &weight, const OptTensor &bias, int64_t num_groups,
                    int64_t activation, double eps) {
    if (!recorded(x, weight, bias)) {
        at::AutoDispatchBelowAutograd guard;
        return op_group_norm().redispatch(below(ks), x, weight, bias, num_groups, activation, eps);
    }
    auto r = GroupNorm::apply(ks, x, weight, bias, num_groups, activation, eps);
    return {r[0], r[1].detach()};
}

struct RelativeBias : torch::autograd::Function<RelativeBias> {
    static constexpr bool is_traceable = true;
    static Tensor forward(AutogradContext *ctx, DispatchKeySet ks, const Tensor &weight, const Tensor &buckets,
                          const OptTensor &starts, SymInt q_len, SymInt k_len, SymInt offset, bool causal,
                          at::ScalarType output_dtype) {
        at::AutoDispatchBelowAutograd guard;
        Tensor out = op_relative_bias().redispatch(below(ks), weight, buckets, starts, q_len, k_len, offset, causal,
                                                   output_dtype);
        ctx->save_for_backward({buckets, starts.value_or(Tensor())});
        ctx->saved_data["rows"] = weight.sym_size(0);
        ctx->saved_data["offset"] = offset;
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["dtype"] = static_cast<int64_t>(weight.scalar_type());
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        variable_list r(9);
        if (!grads[0].defined()) return r;
        const auto s = ctx->get_saved_variables();
        r[1] = op_relative_bias_backward().call(grads[0].contiguous(), s[0], maybe(s[1]), ctx->saved_data["rows"].toSymInt(),
                                                ctx->saved_data["offset"].toSymInt(), ctx->saved_data["causal"].toBool(),
                                                static_cast<at::ScalarType>(ctx->saved_data["dtype"].toInt()));
        return r;
    }
};

// (lengths, the offset and the table's rows are symbols where a graph is made for all of them)
Tensor relative_bias(DispatchKeySet ks, const Tensor &weight, const Tensor &buckets, const OptTensor &starts, SymInt q_len,
                     SymInt k_len, SymInt offset, bool causal, at::ScalarType output_dtype) {
    if (!recorded(weight)) {
        at::AutoDispatchBelowAutograd guard;
        return op_relative_bias().redispatch(below(ks), weight, buckets, starts, q_len, k_len, offset, causal, output_dtype);
    }
    return RelativeBias::apply(ks, weight, buckets, starts, q_len, k_len, offset, causal, output_dtype);
}

}  // namespace

TORCH_LIBRARY_IMPL(rtdl_num_embeddings_cuda, Autograd, m) {
    m.impl("group_norm", TORCH_FN(group_norm));
    m.impl("relative_bias", TORCH_FN(relative_bias));
    m.impl("gradient_norm", torch::CppFunction::makeFallthrough());
    m.impl("clip_gradients_", torch::CppFunction::makeFallthrough());
    m.impl("clip_gradients_into", torch::CppFunction::makeFallthrough());
}

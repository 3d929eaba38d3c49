// What the autograd formulas share: typed operator handles, which inputs are
// recorded, and which gradients are wanted.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <tuple>

namespace {

using at::Tensor;
using c10::DispatchKeySet;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

template <typename Sig>
c10::TypedOperatorHandle<Sig> find_op(const char *name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}

#define PLE_OP(fn, name, ...)                                                                   \
    const c10::TypedOperatorHandle<__VA_ARGS__> &fn() {                                         \
        static const auto op = find_op<__VA_ARGS__>("rtdl_num_embeddings_cuda::" name);         \
        return op;                                                                              \
    }

bool wants(const Tensor &t) { return t.defined() && t.requires_grad(); }
bool wants(const OptTensor &t) { return t.has_value() && wants(*t); }

bool has_tangent(const Tensor &t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool has_tangent(const OptTensor &t) { return t.has_value() && has_tangent(*t); }

// whether the call is recorded: grad mode, and an input that requires grad
template <typename... T>
bool recorded(const T &...t) {
    if (!at::GradMode::is_enabled() || !(wants(t) || ...)) return false;
    TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(t) || ...), "The PLE operators have no forward-mode derivative.");
    return true;
}

DispatchKeySet below(DispatchKeySet ks) { return ks & c10::after_autograd_keyset; }

// bit i: gradient i is wanted
template <typename... T>
int64_t need_bits(const T &...t) {
    int64_t bits = 0, i = 0;
    ((bits |= static_cast<int64_t>(wants(t)) << i++), ...);
    return bits;
}

Tensor if_bit(int64_t bits, int i, Tensor t) { return (bits >> i) & 1 ? std::move(t) : Tensor(); }

}  // namespace

// PyTorch dispatcher registration of group_norm, relative_bias (each with its
// backward) and of the gradients' norm and clipping.  Host code only, as
// ple_token_ops.cpp: it validates the tensors, allocates outputs and scratch with
// the ATen caching allocator, and calls the C ABI of include/ple_hip.h on the
// caller's current HIP stream, without a host synchronisation.

#include <ATen/MemoryOverlap.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <tuple>
#include <utility>
#include <vector>

#include "ple_torch.h"

namespace {

using at::Tensor;
using OptTensor = c10::optional<Tensor>;

bool is_float_type(at::ScalarType t) { return ple_dtype_of(t) >= 0; }

void check_tensor(const Tensor &t, const Tensor &like, const char *name) {
    TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on the same CUDA device as the other tensors");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

bool has(const OptTensor &t) { return t.has_value() && t->defined(); }

const void *opt_ptr(const OptTensor &t) { return has(t) ? t->data_ptr() : nullptr; }

Tensor scratch(size_t bytes, const Tensor &like) {
    return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

// ---------------------------------------------------------------------------
// group norm
// ---------------------------------------------------------------------------

struct GroupSizes {
    int64_t N, S, C;
    int param_dtype;
};

GroupSizes check_group(const Tensor &x, const OptTensor &weight, const OptTensor &bias, int64_t num_groups,
                       int64_t activation) {
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    check_tensor(x, x, "x");
    TORCH_CHECK(x.dim() >= 2 && x.size(-1) > 0, "x must have shape [N, ..., C]");
    TORCH_CHECK(is_float_type(x.scalar_type()), "x must be float32, float16, or bfloat16");
    TORCH_CHECK(num_groups > 0 && x.size(-1) % num_groups == 0, "num_groups must divide the number of channels, got ",
                num_groups, " and ", x.size(-1));
    TORCH_CHECK(activation >= 0 && activation <= 3, "activation must be 0 (none), 1 (relu), 2 (silu) or 3 (gelu)");
    GroupSizes s{x.size(0), 1, x.size(-1), PLE_DTYPE_F32};
    for (int64_t i = 1; i + 1 < x.dim(); ++i) s.S *= x.size(i);
    for (const auto &[t, name] : {std::pair<const OptTensor &, const char *>{weight, "weight"}, {bias, "bias"}}) {
        if (!has(t)) continue;
        check_tensor(*t, x, name);
        TORCH_CHECK(is_float_type(t->scalar_type()), name, " must be float32, float16, or bfloat16");
        TORCH_CHECK(t->dim() == 1 && t->size(0) == s.C, name, " must have shape [C]");
        s.param_dtype = ple_dtype_of(t->scalar_type());
    }
    TORCH_CHECK(!has(weight) || !has(bias) || weight->scalar_type() == bias->scalar_type(),
                "weight and bias must have one dtype");
    return s;
}

std::tuple<Tensor, Tensor> ple_group_norm(const Tensor &x, const OptTensor &weight, const OptTensor &bias,
                                          int64_t num_groups, int64_t activation, double eps) {
    const GroupSizes s = check_group(x, weight, bias, num_groups, activation);
    DeviceScope scope(x.device().index());
    Tensor y = at::empty_like(x);
    Tensor stats = at::empty({s.N, num_groups, 2}, x.options().dtype(at::kFloat));
    if (x.numel() == 0) return {y, stats.zero_()};
    const int dtype = ple_dtype_of(x.scalar_type());
    const size_t bytes = ple_group_norm_workspace_bytes(s.N, s.S, s.C, num_groups, dtype);
    Tensor ws;
    if (bytes > 0) ws = scratch(bytes, x);
    const int rc = ple_group_norm_launch(x.data_ptr(), opt_ptr(weight), opt_ptr(bias), y.data_ptr(), stats.data_ptr<float>(),
                                         s.N, s.S, s.C, num_groups, static_cast<int>(activation), static_cast<float>(eps),
                                         dtype, s.param_dtype, bytes > 0 ? ws.data_ptr() : nullptr, bytes, current_stream(x));
    check_rc(rc, "ple_group_norm_launch");
    return {y, stats};
}

std::tuple<Tensor, Tensor, Tensor> ple_group_norm_backward(const Tensor &grad_y, const Tensor &x, const Tensor &stats,
                                                           const OptTensor &weight, const OptTensor &bias,
                                                           int64_t num_groups, int64_t activation,
                                                           std::array<bool, 3> output_mask) {
    const GroupSizes s = check_group(x, weight, bias, num_groups, activation);
    check_tensor(grad_y, x, "grad_y");
    TORCH_CHECK(grad_y.sizes() == x.sizes() && grad_y.scalar_type() == x.scalar_type(),
                "grad_y must have the shape and dtype of x");
    check_tensor(stats, x, "stats");
    TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.dim() == 3 && stats.size(0) == s.N &&
                    stats.size(1) == num_groups && stats.size(2) == 2,
                "stats must be the float32 [N, G, 2] of the forward");
    DeviceScope scope(x.device().index());
    void *gx = nullptr, *gw = nullptr, *gb = nullptr;
    const auto out = [&](bool wanted, const OptTensor &like, void *&p) {
        if (!wanted || !has(like)) return at::empty({0}, x.options());
        Tensor t = at::empty_like(*like);
        p = t.data_ptr();
        return t;
    };
    Tensor grad_x = out(output_mask[0], x, gx);
    Tensor grad_weight = out(output_mask[1], weight, gw);
    Tensor grad_bias = out(output_mask[2], bias, gb);
    const int dtype = ple_dtype_of(x.scalar_type());
    const size_t bytes = ple_group_norm_backward_workspace_bytes(s.N, s.S, s.C, num_groups, dtype);
    Tensor ws;
    if (bytes > 0) ws = scratch(bytes, x);
    const int rc = ple_group_norm_backward_launch(grad_y.data_ptr(), x.data_ptr(), stats.data_ptr<float>(), opt_ptr(weight),
                                                  opt_ptr(bias), gx, gw, gb, s.N, s.S, s.C, num_groups,
                                                  static_cast<int>(activation), dtype, s.param_dtype,
                                                  bytes > 0 ? ws.data_ptr() : nullptr, bytes, current_stream(x));
    check_rc(rc, "ple_group_norm_backward_launch");
    return {grad_x, grad_weight, grad_bias};
}

// ---------------------------------------------------------------------------
// relative bias
// ---------------------------------------------------------------------------

int64_t check_bias(const Tensor &buckets, const OptTensor &starts, const Tensor &like) {
    check_tensor(buckets, like, "buckets");
    TORCH_CHECK(buckets.scalar_type() == at::kInt && buckets.dim() == 1 && buckets.size(0) >= 3 && buckets.size(0) % 2 == 1,
                "buckets must be int32 [2 * far + 1], far at least 1");
    if (has(starts)) {
        check_tensor(*starts, like, "starts");
        TORCH_CHECK(starts->scalar_type() == at::kLong && starts->dim() == 1, "starts must be int64 [B]");
    }
    return buckets.size(0) / 2;
}

Tensor ple_relative_bias(const Tensor &weight, const Tensor &buckets, const OptTensor &starts, int64_t q_len, int64_t k_len,
                         int64_t offset, bool causal, at::ScalarType output_dtype) {
    TORCH_CHECK(weight.is_cuda(), "weight must be a CUDA tensor");
    check_tensor(weight, weight, "weight");
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0, "weight must have shape [R, H]");
    TORCH_CHECK(is_float_type(weight.scalar_type()), "weight must be float32, float16, or bfloat16");
    TORCH_CHECK(is_float_type(output_dtype), "output_dtype must be float32, float16, or bfloat16");
    TORCH_CHECK(q_len >= 0 && k_len >= 0, "q_len and k_len must not be negative, got ", q_len, " and ", k_len);
    const int64_t far = check_bias(buckets, starts, weight), R = weight.size(0), H = weight.size(1);
    const int64_t B = has(starts) ? starts->size(0) : 1;
    DeviceScope scope(weight.device().index());
    at::DimVector shape;
    if (has(starts)) shape.push_back(B);
    for (int64_t n : {H, q_len, k_len}) shape.push_back(n);
    Tensor out = at::empty(shape, weight.options().dtype(output_dtype));
    if (out.numel() == 0) return out;
    const int rc = ple_relative_bias_launch(weight.data_ptr(), buckets.data_ptr<int32_t>(),
                                            static_cast<const int64_t *>(opt_ptr(starts)), out.data_ptr(), B, H, q_len,
                                            k_len, R, far, offset, causal, ple_dtype_of(weight.scalar_type()),
                                            ple_dtype_of(output_dtype), current_stream(weight));
    check_rc(rc, "ple_relative_bias_launch");
    return out;
}

Tensor ple_relative_bias_backward(const Tensor &grad_output, const Tensor &buckets, const OptTensor &starts,
                                  int64_t num_rows, int64_t offset, bool causal, at::ScalarType grad_dtype) {
    TORCH_CHECK(grad_output.is_cuda(), "grad_output must be a CUDA tensor");
    check_tensor(grad_output, grad_output, "grad_output");
    const int64_t far = check_bias(buckets, starts, grad_output), lead = has(starts) ? 1 : 0;
    TORCH_CHECK(grad_output.dim() == 3 + lead && grad_output.size(lead) > 0 && (!lead || grad_output.size(0) == starts->size(0)),
                "grad_output must have shape [H, q, k], or [B, H, q, k] with starts");
    TORCH_CHECK(is_float_type(grad_output.scalar_type()), "grad_output must be float32, float16, or bfloat16");
    TORCH_CHECK(is_float_type(grad_dtype), "grad_dtype must be float32, float16, or bfloat16");
    TORCH_CHECK(num_rows > 0, "num_rows must be positive");
    const int64_t B = lead ? grad_output.size(0) : 1, H = grad_output.size(lead), q = grad_output.size(lead + 1),
                  k = grad_output.size(lead + 2);
    DeviceScope scope(grad_output.device().index());
    Tensor grad_weight = at::empty({num_rows, H}, grad_output.options().dtype(grad_dtype));
    const size_t bytes = ple_relative_bias_backward_workspace_bytes(B, H, q, k, num_rows, far);
    Tensor ws;
    if (bytes > 0) ws = scratch(bytes, grad_output);
    const int rc = ple_relative_bias_backward_launch(
        grad_output.data_ptr(), buckets.data_ptr<int32_t>(), static_cast<const int64_t *>(opt_ptr(starts)),
        grad_weight.data_ptr(), B, H, q, k, num_rows, far, offset, causal, ple_dtype_of(grad_output.scalar_type()),
        ple_dtype_of(grad_dtype), bytes > 0 ? ws.data_ptr() : nullptr, bytes, current_stream(grad_output));
    check_rc(rc, "ple_relative_bias_backward_launch");
    return grad_weight;
}

// ---------------------------------------------------------------------------
// the norm of many gradients, and their clipping
// ---------------------------------------------------------------------------

int norm_kind(double norm_type) {
    if (norm_type == 2.0) return PLE_NORM_P2;
    if (norm_type == 1.0) return PLE_NORM_P1;
    TORCH_CHECK(std::isinf(norm_type) && norm_type > 0, "norm_type must be 1, 2 or infinity, got ", norm_type);
    return PLE_NORM_INF;
}

// The list of a call; `out`: where the scaled gradients go.  Elements are taken in
// the order in which they lie in memory, which both sides have to share; a gradient
// with gaps or overlaps is read from a copy, kept in `copies`.
struct Listed {
    std::vector<ple_grad_t> grads;
    std::vector<std::pair<size_t, Tensor>> copies;
};

Listed describe(at::TensorList grads, const at::TensorList *out) {
    TORCH_CHECK(!grads.empty(), "there has to be a gradient");
    TORCH_CHECK(!out || out->size() == grads.size(), "out must have a tensor for every gradient");
    Listed list;
    list.grads.reserve(grads.size());
    const c10::Device device = grads[0].device();
    const auto check = [&](const Tensor &t, const char *name) {
        TORCH_CHECK(t.is_cuda() && t.device() == device, name, " must be on one CUDA device");
        TORCH_CHECK(t.layout() == at::kStrided, name, " must not be sparse");
        TORCH_CHECK(is_float_type(t.scalar_type()), name, " must be float32, float16, or bfloat16");
    };
    for (size_t i = 0; i < grads.size(); ++i) {
        Tensor g = grads[i];
        check(g, "gradients");
        if (!g.is_non_overlapping_and_dense()) {
            g = g.contiguous();
            list.copies.emplace_back(i, g);
        }
        const int dtype = ple_dtype_of(g.scalar_type());
        ple_grad_t d{g.data_ptr(), g.data_ptr(), g.numel(), dtype, dtype};
        if (out) {
            const Tensor &o = (*out)[i];
            check(o, "out");
            TORCH_CHECK(o.is_non_overlapping_and_dense(), "out must be dense in memory");
            TORCH_CHECK(o.sizes() == g.sizes() && (o.strides() == g.strides() || (o.is_contiguous() && g.is_contiguous())),
                        "out must have the shape and strides of its gradient");
            d.out = o.data_ptr();
            d.out_dtype = ple_dtype_of(o.scalar_type());
        }
        list.grads.push_back(d);
    }
    return list;
}

size_t bytes_of(int dtype) { return dtype == PLE_DTYPE_F32 ? 4 : 2; }

struct Range {
    uintptr_t begin, end;
    bool written;
};

// Whether a range that is written has bytes of another.
bool overlap(std::vector<Range> ranges) {
    std::sort(ranges.begin(), ranges.end(), [](const Range &a, const Range &b) { return a.begin < b.begin; });
    uintptr_t written = 0, read = 0;         // ends of what has been seen
    for (const Range &r : ranges) {
        if (r.begin < written || (r.written && r.begin < read)) return true;
        (r.written ? written : read) = std::max(r.written ? written : read, r.end);
    }
    return false;
}

// A tensor's elements as ranges of memory: all of it, gaps and all, or its runs.
void add_ranges(const Tensor &t, bool runs, std::vector<Range> &ranges) {
    const auto begin = reinterpret_cast<uintptr_t>(t.data_ptr());
    std::vector<std::pair<int64_t, int64_t>> dims;          // stride, size
    for (int64_t k = 0; k < t.dim(); ++k)
        if (t.size(k) > 1) dims.emplace_back(t.stride(k), t.size(k));
    std::sort(dims.begin(), dims.end());
    int64_t run = 1, last = 0;
    size_t inner = 0;
    while (inner < dims.size() && dims[inner].first == run) run *= dims[inner++].second;
    for (const auto &[stride, size] : dims) last += stride * (size - 1);
    const auto push = [&](int64_t first, int64_t n) {
        ranges.push_back({begin + first * t.element_size(), begin + (first + n) * t.element_size(), true});
    };
    if (!runs) return push(0, last + 1);
    std::vector<int64_t> at(dims.size(), 0);
    for (int64_t first = 0;;) {
        push(first, run);
        size_t k = inner;
        for (; k < dims.size(); ++k) {
            first += dims[k].first;
            if (++at[k] < dims[k].second) break;
            first -= dims[k].first * dims[k].second;
            at[k] = 0;
        }
        if (k == dims.size()) return;
    }
}

// Every element is written once, and read by nothing but the one that writes it.
// Gradients with gaps that are scaled in place lie between others, often (columns of
// one tensor): their runs are looked at if they do.
void check_overlap(const Listed &list, at::TensorList grads, bool in_place) {
    std::vector<Range> ranges;
    ranges.reserve(2 * list.grads.size());
    const auto dense = [&] {
        ranges.clear();
        for (const ple_grad_t &g : list.grads) {
            if (g.numel == 0) continue;
            const auto o = reinterpret_cast<uintptr_t>(g.out), p = reinterpret_cast<uintptr_t>(g.grad);
            ranges.push_back({o, o + g.numel * bytes_of(g.out_dtype), true});
            if (o != p) ranges.push_back({p, p + g.numel * bytes_of(g.dtype), false});
            TORCH_CHECK(o != p || g.dtype == g.out_dtype, "a gradient that is scaled in place keeps its dtype");
        }
    };
    const auto all = [&](bool runs) {
        dense();
        for (const auto &[i, copy] : list.copies) {
            if (!in_place || grads[i].numel() == 0) continue;
            at::assert_no_internal_overlap(grads[i]);
            add_ranges(grads[i], runs, ranges);
        }
        return overlap(ranges);
    };
    TORCH_CHECK(!all(false) || (in_place && !list.copies.empty() && !all(true)),
                "gradients that are scaled must not share memory with each other or with out");
}

void check_limit(double max_norm) { TORCH_CHECK(max_norm >= 0, "max_norm must not be negative, got ", max_norm); }

void check_norm(const Tensor &norm, const Tensor &like) {
    check_tensor(norm, like, "norm");
    TORCH_CHECK(norm.scalar_type() == at::kFloat && norm.numel() == 1, "norm must be one float32 value");
}

Tensor ple_gradient_norm(at::TensorList grads, double norm_type) {
    const Listed list = describe(grads, nullptr);
    const int kind = norm_kind(norm_type);
    DeviceScope scope(grads[0].device().index());
    Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
    const int64_t count = static_cast<int64_t>(list.grads.size());
    const size_t bytes = ple_grad_norm_workspace_bytes(list.grads.data(), count);
    Tensor ws = scratch(bytes, grads[0]);
    check_rc(ple_grad_norm_launch(list.grads.data(), count, kind, norm.data_ptr<float>(), ws.data_ptr(), bytes,
                                  current_stream(grads[0])),
             "ple_grad_norm_launch");
    return norm;
}

Tensor clip(at::TensorList grads, const at::TensorList *out, double max_norm, double norm_type, const OptTensor &given) {
    check_limit(max_norm);
    const int kind = norm_kind(norm_type);
    const Listed list = describe(grads, out);
    check_overlap(list, grads, !out);
    if (has(given)) check_norm(*given, grads[0]);
    DeviceScope scope(grads[0].device().index());
    Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
    const int64_t count = static_cast<int64_t>(list.grads.size());
    const float limit = static_cast<float>(max_norm);
    if (has(given)) {
        norm.copy_(given->reshape({}));
        check_rc(ple_grad_scale_launch(list.grads.data(), count, norm.data_ptr<float>(), limit, current_stream(grads[0])),
                 "ple_grad_scale_launch");
    } else {
        const size_t bytes = ple_grad_norm_workspace_bytes(list.grads.data(), count);
        Tensor ws = scratch(bytes, grads[0]);
        check_rc(ple_grad_clip_launch(list.grads.data(), count, kind, limit, norm.data_ptr<float>(), ws.data_ptr(), bytes,
                                      current_stream(grads[0])),
                 "ple_grad_clip_launch");
    }
    if (!out)
        for (const auto &[i, copy] : list.copies) grads[i].copy_(copy);
    // (what autograd has saved of them is no longer there)
    for (const Tensor &t : out ? *out : grads)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    return norm;
}

Tensor ple_clip_gradients_(at::TensorList grads, double max_norm, double norm_type, const OptTensor &norm) {
    return clip(grads, nullptr, max_norm, norm_type, norm);
}

Tensor ple_clip_gradients_into(at::TensorList grads, at::TensorList out, double max_norm, double norm_type,
                               const OptTensor &norm) {
    return clip(grads, &out, max_norm, norm_type, norm);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(rtdl_num_embeddings_cuda, m) {
    m.def(
        "group_norm(Tensor x, Tensor? weight, Tensor? bias, int num_groups, int activation, float eps) "
        "-> (Tensor y, Tensor stats)");
    m.def(
        "group_norm_backward(Tensor grad_y, Tensor x, Tensor stats, Tensor? weight, Tensor? bias, int num_groups, "
        "int activation, bool[3] output_mask) -> (Tensor grad_x, Tensor grad_weight, Tensor grad_bias)");
    m.def(
        "relative_bias(Tensor weight, Tensor buckets, Tensor? starts, SymInt q_len, SymInt k_len, SymInt offset, bool causal, "
        "ScalarType output_dtype) -> Tensor");
    m.def(
        "relative_bias_backward(Tensor grad_output, Tensor buckets, Tensor? starts, SymInt num_rows, SymInt offset, "
        "bool causal, ScalarType grad_dtype) -> Tensor");
    m.def("gradient_norm(Tensor[] grads, float norm_type) -> Tensor");
    m.def("clip_gradients_(Tensor(a!)[] grads, float max_norm, float norm_type, Tensor? norm) -> Tensor");
    m.def("clip_gradients_into(Tensor[] grads, Tensor(a!)[] out, float max_norm, float norm_type, Tensor? norm) -> Tensor");
}

TORCH_LIBRARY_IMPL(rtdl_num_embeddings_cuda, CUDA, m) {
    m.impl("group_norm", &ple_group_norm);
    m.impl("group_norm_backward", &ple_group_norm_backward);
    m.impl("relative_bias", &ple_relative_bias);
    m.impl("relative_bias_backward", &ple_relative_bias_backward);
    m.impl("gradient_norm", &ple_gradient_norm);
    m.impl("clip_gradients_", &ple_clip_gradients_);
    m.impl("clip_gradients_into", &ple_clip_gradients_into);
}

// The extern "C" entry points of the group norm, the relative position bias and
// the gradients' norm and scaling: argument checks that need no device, then the
// launchers.

#include <cmath>

#include "ple_internal.h"

namespace ple {
namespace {

constexpr int64_t kMaxElems = int64_t{1} << 44;
constexpr int64_t kMaxCount = INT32_MAX;          // rows, samples, heads
constexpr int64_t kMaxChannels = 1 << 20;
constexpr int64_t kMaxFar = 1 << 24;
constexpr int64_t kMaxOffset = int64_t{1} << 60;
constexpr int64_t kMaxLength = 1 << 23;           // (a row block's offsets are 32-bit)

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

bool aligned_for(const void *p, int dtype) { return aligned(p, dtype == PLE_DTYPE_F32 ? 4 : 2); }

bool product_fits(std::initializer_list<int64_t> sizes) {
    int64_t all = 1;
    for (int64_t s : sizes) {
        if (s == 0) return true;
        if (all > kMaxElems / s) return false;
        all *= s;
    }
    return true;
}

int check_group(int64_t N, int64_t S, int64_t C, int64_t G, int dtype) {
    if (N < 0 || S < 0 || C < 1 || G < 1 || C % G != 0) return PLE_E_BAD_SHAPE;
    if (N > kMaxCount || S > kMaxCount || C > kMaxChannels || !product_fits({N, S, C})) return PLE_E_TOO_LARGE;
    return valid_dtype(dtype) ? PLE_OK : PLE_E_BAD_DTYPE;
}

GroupRequest group_request(int64_t N, int64_t S, int64_t C, int64_t G, int dtype) {
    GroupRequest r{};
    r.N = N; r.S = S; r.C = C; r.G = G;
    r.dtype = dtype; r.param_dtype = PLE_DTYPE_F32;
    return r;
}

int check_bias(int64_t B, int64_t H, int64_t q, int64_t k, int64_t R, int64_t far, int64_t offset, bool starts) {
    if (B < 0 || H < 1 || q < 0 || k < 0 || R < 1 || far < 1 || (!starts && B != 1)) return PLE_E_BAD_SHAPE;
    if (B > kMaxCount || H > kMaxCount || q > kMaxLength || k > kMaxLength || R > kMaxCount || far > kMaxFar ||
        offset > kMaxOffset || offset < -kMaxOffset || !product_fits({B, H, q, k}) || !product_fits({R, H}))
        return PLE_E_TOO_LARGE;
    return PLE_OK;
}

int check_grads(const ple_grad_t *grads, int64_t count, bool scaling) {
    if (count < 0) return PLE_E_BAD_SHAPE;
    if (count > 0 && !grads) return PLE_E_NULL_POINTER;
    for (int64_t i = 0; i < count; ++i) {
        const ple_grad_t &g = grads[i];
        if (g.numel < 0) return PLE_E_BAD_SHAPE;
        if (g.numel > (int64_t{1} << 40)) return PLE_E_TOO_LARGE;
        if (!valid_dtype(g.dtype) || (scaling && !valid_dtype(g.out_dtype))) return PLE_E_BAD_DTYPE;
        if (g.numel == 0) continue;
        if (!g.grad || (scaling && !g.out)) return PLE_E_NULL_POINTER;
        if (!aligned_for(g.grad, g.dtype) || (scaling && !aligned_for(g.out, g.out_dtype))) return PLE_E_MISALIGNED;
        if (scaling && g.out == g.grad && g.dtype != g.out_dtype) return PLE_E_UNSUPPORTED;
    }
    return PLE_OK;
}

}  // namespace
}  // namespace ple

extern "C" {

size_t ple_group_norm_workspace_bytes(int64_t N, int64_t S, int64_t C, int64_t G, int dtype) {
    if (ple::check_group(N, S, C, G, dtype) != PLE_OK || N == 0 || S == 0) return 0;
    return ple::group_workspace_bytes(ple::group_request(N, S, C, G, dtype));
}

int ple_group_norm_launch(const void *x, const void *weight, const void *bias, void *y, float *stats, int64_t N,
                          int64_t S, int64_t C, int64_t G, int activation, float eps, int dtype, int param_dtype,
                          void *workspace, size_t workspace_bytes, void *stream) {
    const int rc = ple::check_group(N, S, C, G, dtype);
    if (rc != PLE_OK) return rc;
    if (!ple::valid_dtype(param_dtype)) return PLE_E_BAD_DTYPE;
    if (activation < PLE_ACT_NONE || activation > PLE_ACT_GELU) return PLE_E_UNSUPPORTED;
    if (N == 0 || S == 0) return PLE_OK;
    if (!x || !y || !stats) return PLE_E_NULL_POINTER;
    if (!ple::aligned_for(x, dtype) || !ple::aligned_for(y, dtype) || !ple::aligned(stats, 8) ||
        !ple::aligned_for(weight, param_dtype) || !ple::aligned_for(bias, param_dtype))
        return PLE_E_MISALIGNED;
    ple::GroupRequest r = ple::group_request(N, S, C, G, dtype);
    r.x = x; r.weight = weight; r.bias = bias; r.y = y; r.stats = stats;
    r.param_dtype = param_dtype; r.act = activation; r.eps = eps;
    r.workspace = workspace; r.workspace_bytes = workspace_bytes;
    r.stream = static_cast<hipStream_t>(stream);
    return ple::group_run(r);
}

size_t ple_group_norm_backward_workspace_bytes(int64_t N, int64_t S, int64_t C, int64_t G, int dtype) {
    if (ple::check_group(N, S, C, G, dtype) != PLE_OK || N == 0 || S == 0) return 0;
    return ple::group_backward_workspace_bytes(ple::group_request(N, S, C, G, dtype));
}

int ple_group_norm_backward_launch(const void *grad_y, const void *x, const float *stats, const void *weight,
                                   const void *bias, void *grad_x, void *grad_weight, void *grad_bias, int64_t N,
                                   int64_t S, int64_t C, int64_t G, int activation, int dtype, int param_dtype,
                                   void *workspace, size_t workspace_bytes, void *stream) {
    const int rc = ple::check_group(N, S, C, G, dtype);
    if (rc != PLE_OK) return rc;
    if (!ple::valid_dtype(param_dtype)) return PLE_E_BAD_DTYPE;
    if (activation < PLE_ACT_NONE || activation > PLE_ACT_GELU) return PLE_E_UNSUPPORTED;
    if (!grad_x && !grad_weight && !grad_bias) return PLE_OK;
    if (N > 0 && S > 0 && (!grad_y || !x || !stats)) return PLE_E_NULL_POINTER;
    for (const void *p : {grad_y, x, static_cast<const void *>(grad_x)})
        if (!ple::aligned_for(p, dtype)) return PLE_E_MISALIGNED;
    for (const void *p : {weight, bias, static_cast<const void *>(grad_weight), static_cast<const void *>(grad_bias)})
        if (!ple::aligned_for(p, param_dtype)) return PLE_E_MISALIGNED;
    if (!ple::aligned(stats, 8)) return PLE_E_MISALIGNED;
    ple::GroupRequest r = ple::group_request(N, S, C, G, dtype);
    r.x = x; r.weight = weight; r.bias = bias; r.g = grad_y; r.y = grad_x;
    r.d_weight = grad_weight; r.d_bias = grad_bias;
    r.stats = const_cast<float *>(stats);
    r.param_dtype = param_dtype; r.act = activation;
    r.workspace = workspace; r.workspace_bytes = workspace_bytes;
    r.stream = static_cast<hipStream_t>(stream);
    return ple::group_backward_run(r);
}

int ple_group_norm_plan_query(const void *x, int64_t N, int64_t S, int64_t C, int64_t G, int dtype, int backward,
                              ple_group_norm_plan_info_t *info) {
    const int rc = ple::check_group(N, S, C, G, dtype);
    if (rc != PLE_OK) return rc;
    if (!info) return PLE_E_NULL_POINTER;
    ple::GroupRequest r = ple::group_request(N, S, C, G, dtype);
    r.x = x;
    return ple::group_plan_info(r, backward != 0, info);
}

int ple_relative_bias_launch(const void *weight, const int32_t *buckets, const int64_t *starts, void *out, int64_t B,
                             int64_t H, int64_t q, int64_t k, int64_t R, int64_t far, int64_t offset, int causal,
                             int weight_dtype, int out_dtype, void *stream) {
    const int rc = ple::check_bias(B, H, q, k, R, far, offset, starts != nullptr || B == 0);
    if (rc != PLE_OK) return rc;
    if (!ple::valid_dtype(weight_dtype) || !ple::valid_dtype(out_dtype)) return PLE_E_BAD_DTYPE;
    if (B == 0 || q == 0 || k == 0) return PLE_OK;
    if (!weight || !buckets || !out) return PLE_E_NULL_POINTER;
    if (!ple::aligned_for(weight, weight_dtype) || !ple::aligned_for(out, out_dtype) || !ple::aligned(buckets, 4) ||
        !ple::aligned(starts, 8))
        return PLE_E_MISALIGNED;
    ple::BiasRequest r{};
    r.weight = weight; r.buckets = buckets; r.starts = starts; r.out = out;
    r.B = B; r.H = H; r.q = q; r.k = k; r.R = R; r.far = far; r.offset = offset;
    r.causal = causal != 0; r.weight_dtype = weight_dtype; r.out_dtype = out_dtype;
    r.stream = static_cast<hipStream_t>(stream);
    return ple::bias_run(r);
}

size_t ple_relative_bias_backward_workspace_bytes(int64_t B, int64_t H, int64_t q, int64_t k, int64_t R, int64_t far) {
    if (ple::check_bias(B, H, q, k, R, far, 0, true) != PLE_OK) return 0;
    ple::BiasRequest r{};
    r.B = B; r.H = H; r.q = q; r.k = k; r.R = R; r.far = far;
    return ple::bias_backward_workspace_bytes(r);
}

int ple_relative_bias_backward_launch(const void *grad_output, const int32_t *buckets, const int64_t *starts,
                                      void *grad_weight, int64_t B, int64_t H, int64_t q, int64_t k, int64_t R,
                                      int64_t far, int64_t offset, int causal, int out_dtype, int weight_dtype,
                                      void *workspace, size_t workspace_bytes, void *stream) {
    const int rc = ple::check_bias(B, H, q, k, R, far, offset, starts != nullptr || B == 0);
    if (rc != PLE_OK) return rc;
    if (!ple::valid_dtype(weight_dtype) || !ple::valid_dtype(out_dtype)) return PLE_E_BAD_DTYPE;
    if (!grad_weight || !buckets || (B > 0 && q > 0 && k > 0 && !grad_output)) return PLE_E_NULL_POINTER;
    if (!ple::aligned_for(grad_weight, weight_dtype) || !ple::aligned_for(grad_output, out_dtype) ||
        !ple::aligned(buckets, 4) || !ple::aligned(starts, 8))
        return PLE_E_MISALIGNED;
    ple::BiasRequest r{};
    r.grad = grad_output; r.buckets = buckets; r.starts = starts; r.dw = grad_weight;
    r.B = B; r.H = H; r.q = q; r.k = k; r.R = R; r.far = far; r.offset = offset;
    r.causal = causal != 0; r.weight_dtype = weight_dtype; r.out_dtype = out_dtype;
    r.workspace = workspace; r.workspace_bytes = workspace_bytes;
    r.stream = static_cast<hipStream_t>(stream);
    return ple::bias_backward_run(r);
}

size_t ple_grad_norm_workspace_bytes(const ple_grad_t *grads, int64_t count) {
    if (count < 0 || (count > 0 && !grads)) return 0;
    ple::GradsRequest r{};
    r.grads = grads; r.count = count;
    return ple::grad_norm_workspace_bytes(r);
}

int ple_grad_norm_launch(const ple_grad_t *grads, int64_t count, int kind, float *norm, void *workspace,
                         size_t workspace_bytes, void *stream) {
    const int rc = ple::check_grads(grads, count, false);
    if (rc != PLE_OK) return rc;
    if (kind != PLE_NORM_P1 && kind != PLE_NORM_P2 && kind != PLE_NORM_INF) return PLE_E_UNSUPPORTED;
    if (!norm) return PLE_E_NULL_POINTER;
    if (!ple::aligned(norm, 4)) return PLE_E_MISALIGNED;
    ple::GradsRequest r{};
    r.grads = grads; r.count = count; r.kind = kind; r.norm = norm;
    r.workspace = workspace; r.workspace_bytes = workspace_bytes;
    r.stream = static_cast<hipStream_t>(stream);
    return ple::grad_norm_run(r);
}

int ple_grad_scale_launch(const ple_grad_t *grads, int64_t count, const float *norm, float limit, void *stream) {
    const int rc = ple::check_grads(grads, count, true);
    if (rc != PLE_OK) return rc;
    if (!(limit >= 0.0f)) return PLE_E_UNSUPPORTED;
    if (!norm) return PLE_E_NULL_POINTER;
    if (!ple::aligned(norm, 4)) return PLE_E_MISALIGNED;
    ple::GradsRequest r{};
    r.grads = grads; r.count = count; r.norm = const_cast<float *>(norm); r.limit = limit;
    r.stream = static_cast<hipStream_t>(stream);
    return ple::grad_scale_run(r);
}

int ple_grad_clip_launch(const ple_grad_t *grads, int64_t count, int kind, float limit, float *norm, void *workspace,
                         size_t workspace_bytes, void *stream) {
    const int rc = ple::check_grads(grads, count, true);
    if (rc != PLE_OK) return rc;
    if (kind != PLE_NORM_P1 && kind != PLE_NORM_P2 && kind != PLE_NORM_INF) return PLE_E_UNSUPPORTED;
    if (!(limit >= 0.0f)) return PLE_E_UNSUPPORTED;
    if (!norm) return PLE_E_NULL_POINTER;
    if (!ple::aligned(norm, 4)) return PLE_E_MISALIGNED;
    ple::GradsRequest r{};
    r.grads = grads; r.count = count; r.kind = kind; r.norm = norm; r.limit = limit;
    r.workspace = workspace; r.workspace_bytes = workspace_bytes;
    r.stream = static_cast<hipStream_t>(stream);
    return ple::grad_clip_run(r);
}

}  // extern "C"

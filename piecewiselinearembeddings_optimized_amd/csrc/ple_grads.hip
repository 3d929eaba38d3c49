// The norm of many tensors together, and their scaling to a limit (gfx950).
//
//     norm = (sum |g|^p)^(1/p), p = 1 or 2, or max |g|
//     factor = min(1, limit / (norm + 1e-6)),  out = g factor
//
// Bound by memory: a read for the norm; a read and a write for the scaling, which
// does nothing where tensors stay where they are and the factor is 1.  Sums are
// 64-bit: squares of 32-bit values neither overflow nor vanish there, and the
// order of the additions is below the 32-bit result's rounding.  Measured: 54M fp32
// values, norm 43 us (5.0 TB/s), scaling into others 71 us (6.1 TB/s); 354M bf16, norm
// 130 us (5.4 TB/s), scaling into fp32 441 us (4.8 TB/s).
//
// The tensors' addresses and sizes are kernel arguments, kListed of them a launch,
// so a captured graph holds them and nothing is copied to the device.

#include <algorithm>
#include <type_traits>

#include "ple_internal.h"
#include "ple_rows.h"

namespace ple {
namespace {

constexpr int kListed = 100;             // tensors of a launch (its arguments stay below 4 KB)
constexpr int64_t kChunk = 4096;         // elements; workgroups take ranges of chunks
constexpr int kNormThreads = 256;

struct Listed {
    const void *grad;
    void *out;
    int64_t numel;
    int end;                             // chunks of the tensors up to and with this one
    int8_t dtype, out_dtype;
};

struct GradsArgs {
    Listed t[kListed];
    int count, chunks;
    double *partial;                     // of this launch's workgroups; scaling: of the norm's
    float *norm;                         // scaling: read, or written where it has partials
    float limit;
    int kind, partials;                  // scaling: the partials to join (0: the norm is known)
    int in_place;
};
static_assert(sizeof(GradsArgs) <= 4096, "kernel arguments");

// The tensor of a chunk.
__device__ __forceinline__ int find_tensor(const GradsArgs &a, int chunk) {
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (chunk < a.t[mid].end) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// |v| as a value that grows with it, NaN the largest.
__device__ __forceinline__ uint32_t size_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// What a lane has of a norm: a 64-bit sum, or the bits of the largest.
template <int KIND>
struct Norm {
    double sum = 0.0;
    uint32_t most = 0;
    __device__ __forceinline__ void add(float v) {
        if constexpr (KIND == PLE_NORM_P2) sum = fma(static_cast<double>(v), static_cast<double>(v), sum);
        else if constexpr (KIND == PLE_NORM_P1) sum += fabs(static_cast<double>(v));
        else most = max(most, size_bits(v));
    }
    __device__ __forceinline__ void join(const Norm &o) {
        sum += o.sum;
        most = max(most, o.most);
    }
    __device__ __forceinline__ Norm moved(int mask) const {
        Norm o;
        if constexpr (KIND == PLE_NORM_INF) o.most = __shfl_xor(most, mask);
        else o.sum = __shfl_xor(sum, mask);
        return o;
    }
    // over the workgroup, on its first thread
    __device__ __forceinline__ void join_block(double *lds) {
#pragma unroll
        for (int m = 1; m < kWave; m *= 2) join(moved(m));
        if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = packed();
        __syncthreads();
        if (threadIdx.x == 0)
            for (int w = 1; w < static_cast<int>(blockDim.x) / kWave; ++w) add_packed(lds[w]);
    }
    __device__ __forceinline__ double packed() const {
        return KIND == PLE_NORM_INF ? static_cast<double>(__uint_as_float(most)) : sum;
    }
    __device__ __forceinline__ void add_packed(double v) {
        if constexpr (KIND == PLE_NORM_INF) most = max(most, size_bits(static_cast<float>(v)));
        else sum += v;
    }
};

// Elements of 16 bytes, and a type's element from a loaded vector.
template <int T>
constexpr int vec_elems() { return T == PLE_DTYPE_F32 ? 4 : 8; }

template <int T>
__device__ __forceinline__ float vector_elem(const uint4 &raw, int e) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    return grad_elem<T>(w, e);
}

// Elements [begin, end) of p: single ones up to a 16-byte boundary and behind the last,
// vectors between, kFlight of them in flight a lane.
constexpr int kFlight = 8;

template <int T, int KIND>
__device__ __forceinline__ void add_chunk(const void *p, int64_t begin, int64_t end, Norm<KIND> &n) {
    constexpr int E = vec_elems<T>(), kBytes = elem_bytes(T);
    const uint64_t at = reinterpret_cast<uint64_t>(p) / kBytes + begin;
    const int64_t head = min(end, begin + static_cast<int64_t>((E - at % E) % E));
    const int vecs = static_cast<int>((end - head) / E);
    const int64_t tail = head + static_cast<int64_t>(vecs) * E;
    if (threadIdx.x < head - begin) n.add(load_grad<T>(p, begin + threadIdx.x));
    if (threadIdx.x < end - tail) n.add(load_grad<T>(p, tail + threadIdx.x));
    const uint4 *const q = reinterpret_cast<const uint4 *>(static_cast<const char *>(p) + head * kBytes);
    for (int i = threadIdx.x; i < vecs; i += kFlight * kNormThreads) {
        uint4 raw[kFlight];
        // (vectors past the end are read again as the last one, and not added)
#pragma unroll
        for (int v = 0; v < kFlight; ++v) raw[v] = q[min(i + v * kNormThreads, vecs - 1)];
#pragma unroll
        for (int v = 0; v < kFlight; ++v)
            if (i + v * kNormThreads < vecs)
#pragma unroll
                for (int e = 0; e < E; ++e) n.add(vector_elem<T>(raw[v], e));
    }
}

// The workgroup's chunks: an even share of them, in order.
struct Range {
    int begin, end;
    __device__ __forceinline__ explicit Range(const GradsArgs &a) {
        const int each = a.chunks / static_cast<int>(gridDim.x), more = a.chunks - each * static_cast<int>(gridDim.x);
        const int b = static_cast<int>(blockIdx.x);
        begin = b * each + min(b, more);
        end = begin + each + (b < more ? 1 : 0);
    }
};

template <int KIND>
__global__ __launch_bounds__(kNormThreads) void ple_grad_norm_kernel(GradsArgs a) {
    __shared__ double s_norm[kNormThreads / kWave];
    Norm<KIND> n;
    const Range range(a);
    int i = find_tensor(a, range.begin);
    for (int c = range.begin; c < range.end; ++i) {
        const int first = i > 0 ? a.t[i - 1].end : 0, stop = min(range.end, a.t[i].end);
        const int64_t begin = static_cast<int64_t>(c - first) * kChunk;
        const int64_t end = min(a.t[i].numel, static_cast<int64_t>(stop - first) * kChunk);
        if (a.t[i].dtype == PLE_DTYPE_F32) add_chunk<PLE_DTYPE_F32>(a.t[i].grad, begin, end, n);
        else if (a.t[i].dtype == PLE_DTYPE_BF16) add_chunk<PLE_DTYPE_BF16>(a.t[i].grad, begin, end, n);
        else add_chunk<PLE_DTYPE_F16>(a.t[i].grad, begin, end, n);
        c = stop;
    }
    n.join_block(s_norm);
    if (threadIdx.x == 0) a.partial[blockIdx.x] = n.packed();
}

// The norm from the workgroups' partials, in a fixed order, on the first thread.
template <int KIND>
__device__ __forceinline__ float join_partials(const double *partial, int count, double *lds) {
    Norm<KIND> n;
#pragma unroll 4
    for (int i = threadIdx.x; i < count; i += kNormThreads) n.add_packed(partial[i]);
    n.join_block(lds);
    if constexpr (KIND == PLE_NORM_INF) return __uint_as_float(n.most);
    else return static_cast<float>(KIND == PLE_NORM_P2 ? sqrt(n.sum) : n.sum);
}

template <int KIND>
__global__ __launch_bounds__(kNormThreads) void ple_grad_norm_join_kernel(const double *partial, int count, float *norm) {
    __shared__ double s_norm[kNormThreads / kWave];
    const float v = join_partials<KIND>(partial, count, s_norm);
    if (threadIdx.x == 0) *norm = v;
}

// Elements [begin, end) of p times the factor, as type O: from the end on, where caches
// may still have what the norm read last.
template <int T, int O, bool NT>
__device__ __forceinline__ void scale_range(const void *p, void *out, int64_t begin, int64_t end, float factor) {
    // vectors of 16 bytes of out, where both sides have their boundaries at the same
    // elements (a lane's two stores of 16 bytes side by side would leave halves of lines
    // to go past the caches: 355M bf16 into fp32 562 us, 440 through them)
    constexpr int E = vec_elems<O>(), kIn = elem_bytes(T), kOut = elem_bytes(O);
    constexpr int kWords = E * kIn / 4, kSteps = kWords >= 4 ? 16 / kWords : 4;
    const uint64_t at = reinterpret_cast<uint64_t>(out) / kOut + begin, in = reinterpret_cast<uint64_t>(p) / kIn + begin;
    const auto one = [&](int64_t i) {
        const float v = load_grad<T>(p, i) * factor;
        store_vec<O, 1>(out, i, &v);
    };
    if ((at - in) % E != 0) {
        for (int64_t i = end - 1 - threadIdx.x; i >= begin; i -= kNormThreads) one(i);
        return;
    }
    const int64_t head = min(end, begin + static_cast<int64_t>((E - at % E) % E));
    const int vecs = static_cast<int>((end - head) / E);
    const int64_t tail = head + static_cast<int64_t>(vecs) * E;
    if (threadIdx.x < head - begin) one(begin + threadIdx.x);
    if (threadIdx.x < end - tail) one(tail + threadIdx.x);
    if (vecs == 0) return;
    const char *const src = static_cast<const char *>(p) + head * kIn;
    char *const dst = static_cast<char *>(out) + head * kOut;
    constexpr int kTurn = kSteps * kNormThreads;
    for (int i0 = (vecs - 1) / kTurn * kTurn; i0 >= 0; i0 -= kTurn) {
        uint32_t raw[kSteps][kWords];
#pragma unroll
        for (int v = 0; v < kSteps; ++v) {
            const int64_t i = min(i0 + v * kNormThreads + static_cast<int>(threadIdx.x), vecs - 1);
            if constexpr (kWords == 2) {
                const uint2 w = reinterpret_cast<const uint2 *>(src)[i];
                raw[v][0] = w.x; raw[v][1] = w.y;
            } else {
#pragma unroll
                for (int k = 0; k < kWords / 4; ++k) {
                    const uint4 w = reinterpret_cast<const uint4 *>(src)[i * (kWords / 4) + k];
                    raw[v][4 * k] = w.x; raw[v][4 * k + 1] = w.y; raw[v][4 * k + 2] = w.z; raw[v][4 * k + 3] = w.w;
                }
            }
        }
#pragma unroll
        for (int v = 0; v < kSteps; ++v) {
            const int i = i0 + v * kNormThreads + threadIdx.x;
            float f[E];
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = grad_elem<T>(raw[v], e) * factor;
            if (i < vecs) store_vec<O, E, NT>(dst, static_cast<int64_t>(i) * E, f);
        }
    }
}

template <bool NT>
__global__ __launch_bounds__(kNormThreads) void ple_grad_scale_kernel(GradsArgs a) {
    __shared__ double s_norm[kNormThreads / kWave];
    __shared__ float s_joined;
    if (a.partials > 0) {
        float v;
        if (a.kind == PLE_NORM_P2) v = join_partials<PLE_NORM_P2>(a.partial, a.partials, s_norm);
        else if (a.kind == PLE_NORM_P1) v = join_partials<PLE_NORM_P1>(a.partial, a.partials, s_norm);
        else v = join_partials<PLE_NORM_INF>(a.partial, a.partials, s_norm);
        if (threadIdx.x == 0) {
            s_joined = v;
            if (blockIdx.x == 0) *a.norm = v;
        }
        __syncthreads();
    }
    const float norm = a.partials > 0 ? s_joined : *a.norm;
    // (an infinite limit clips nothing; a norm of NaN makes everything NaN)
    const double ratio = static_cast<double>(a.limit) / (static_cast<double>(norm) + 1e-6);
    const float factor = a.limit == __builtin_inff() || ratio >= 1.0 ? 1.0f : static_cast<float>(ratio);
    if (a.in_place && factor == 1.0f) return;
    const Range range(a);
    int i = find_tensor(a, range.end - 1);
    for (int c = range.end; c > range.begin; --i) {
        const Listed &t = a.t[i];
        const int first = i > 0 ? a.t[i - 1].end : 0, from = max(range.begin, first);
        const int64_t begin = static_cast<int64_t>(from - first) * kChunk;
        const int64_t end = min(t.numel, static_cast<int64_t>(c - first) * kChunk);
        const auto to = [&](auto of) {
            constexpr int T = decltype(of)::value;
            if (t.out_dtype == PLE_DTYPE_F32) scale_range<T, PLE_DTYPE_F32, NT>(t.grad, t.out, begin, end, factor);
            else if (t.out_dtype == PLE_DTYPE_BF16) scale_range<T, PLE_DTYPE_BF16, NT>(t.grad, t.out, begin, end, factor);
            else scale_range<T, PLE_DTYPE_F16, NT>(t.grad, t.out, begin, end, factor);
        };
        if (t.dtype == PLE_DTYPE_F32) to(std::integral_constant<int, PLE_DTYPE_F32>{});
        else if (t.dtype == PLE_DTYPE_BF16) to(std::integral_constant<int, PLE_DTYPE_BF16>{});
        else to(std::integral_constant<int, PLE_DTYPE_F16>{});
        c = from;
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

// The tensors of the list from `from` on that one launch takes; returns where the
// next launch begins.  (A launch's chunks are counted in 32 bits.)
int64_t fill(const ple_grad_t *grads, int64_t count, int64_t from, GradsArgs &a) {
    a.count = 0;
    a.chunks = 0;
    a.in_place = 1;
    int64_t i = from;
    for (; i < count && a.count < kListed; ++i) {
        if (grads[i].numel == 0) continue;
        const int64_t chunks = (grads[i].numel + kChunk - 1) / kChunk;
        if (a.chunks + chunks > INT32_MAX / 2) break;        // (numel is below 2^40: one tensor always fits)
        Listed &t = a.t[a.count++];
        t.grad = grads[i].grad;
        t.out = grads[i].out;
        t.numel = grads[i].numel;
        t.dtype = static_cast<int8_t>(grads[i].dtype);
        t.out_dtype = static_cast<int8_t>(grads[i].out_dtype);
        a.chunks += static_cast<int>(chunks);
        t.end = a.chunks;
        if (t.out != t.grad) a.in_place = 0;
    }
    return i;
}

int grid_of(const GradsArgs &a) { return std::min(a.chunks, 8 * device_cu_count()); }

// The norm's partials; their number in `used`.
template <int KIND>
int partial_launches(const GradsRequest &r, int &used) {
    GradsArgs a{};
    used = 0;
    for (int64_t from = 0; from < r.count;) {
        from = fill(r.grads, r.count, from, a);
        if (a.count == 0) break;
        a.partial = static_cast<double *>(r.workspace) + used;
        const int grid = grid_of(a);
        used += grid;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_grad_norm_kernel<KIND>), dim3(grid), dim3(kNormThreads), 0, r.stream, a);
        const hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return static_cast<int>(rc);
    }
    return PLE_OK;
}

template <int KIND>
int join_launch(const GradsRequest &r, int used) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_grad_norm_join_kernel<KIND>), dim3(1), dim3(kNormThreads), 0, r.stream,
                       static_cast<const double *>(r.workspace), used, r.norm);
    return static_cast<int>(hipGetLastError());
}

int partial_launches(const GradsRequest &r, int &used) {
    if (r.kind == PLE_NORM_P2) return partial_launches<PLE_NORM_P2>(r, used);
    if (r.kind == PLE_NORM_P1) return partial_launches<PLE_NORM_P1>(r, used);
    return partial_launches<PLE_NORM_INF>(r, used);
}

int join_launch(const GradsRequest &r, int used) {
    if (r.kind == PLE_NORM_P2) return join_launch<PLE_NORM_P2>(r, used);
    if (r.kind == PLE_NORM_P1) return join_launch<PLE_NORM_P1>(r, used);
    return join_launch<PLE_NORM_INF>(r, used);
}

bool bad_workspace(const GradsRequest &r) {
    return !r.workspace || r.workspace_bytes < grad_norm_workspace_bytes(r) || reinterpret_cast<uintptr_t>(r.workspace) % 256 != 0;
}

}  // namespace

size_t grad_norm_workspace_bytes(const GradsRequest &r) {
    GradsArgs a{};
    int64_t used = 0;
    for (int64_t from = 0; from < r.count;) {
        from = fill(r.grads, r.count, from, a);
        if (a.count == 0) break;
        used += grid_of(a);
    }
    return align_up(static_cast<size_t>(std::max<int64_t>(used, 1)) * 8, 256);
}

int grad_norm_run(const GradsRequest &r) {
    if (bad_workspace(r)) return PLE_E_WORKSPACE;
    int used = 0;
    const int rc = partial_launches(r, used);
    return rc != PLE_OK ? rc : join_launch(r, used);
}

namespace {

// `partials`: the norm's, for the scaling's workgroups to join.
int scale_launches(const GradsRequest &r, int partials) {
    // What the memory-side cache (256 MB) cannot hold is written past the caches, so that
    // the next reads do not wait for it (54M fp32 into fp32, with the norm: 138 us with
    // plain stores, 113 without).
    int64_t bytes = 0;
    for (int64_t i = 0; i < r.count; ++i)
        bytes += r.grads[i].numel * (elem_bytes(r.grads[i].dtype) + (r.grads[i].out != r.grads[i].grad ? elem_bytes(r.grads[i].out_dtype) : 0));
    const bool stream = bytes > (int64_t{256} << 20);
    GradsArgs a{};
    a.norm = r.norm;
    a.limit = r.limit;
    a.kind = r.kind;
    a.partial = static_cast<double *>(r.workspace);
    a.partials = partials;
    for (int64_t from = 0; from < r.count;) {
        from = fill(r.grads, r.count, from, a);
        if (a.count == 0) break;
        if (stream) hipLaunchKernelGGL(ple_grad_scale_kernel<true>, dim3(grid_of(a)), dim3(kNormThreads), 0, r.stream, a);
        else hipLaunchKernelGGL(ple_grad_scale_kernel<false>, dim3(grid_of(a)), dim3(kNormThreads), 0, r.stream, a);
        const hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return static_cast<int>(rc);
    }
    return PLE_OK;
}

}  // namespace

int grad_scale_run(const GradsRequest &r) { return scale_launches(r, 0); }

int grad_clip_run(const GradsRequest &r) {
    if (bad_workspace(r)) return PLE_E_WORKSPACE;
    int used = 0, rc = partial_launches(r, used);
    if (rc != PLE_OK) return rc;
    // As many partials as one launch leaves are joined by every workgroup that scales, not by a
    // launch of its own between (906 k values in 33 tensors: 8.9 us, with it 12.9); more of them
    // would be too much to read again.
    if (used > 0 && used <= 8 * device_cu_count()) return scale_launches(r, used);
    rc = join_launch(r, used);
    return rc != PLE_OK ? rc : scale_launches(r, 0);
}

}  // namespace ple

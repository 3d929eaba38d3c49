// Learned bias of attention scores by relative position (gfx950).  Query i of a
// sample stands at position start + i, key j at j; a table of rows by buckets of
// distances gives every head a value:
//
//     out[h, i, j] = w[row(j - start - i), h],   row(d) = buckets[clamp(d, -M, M) + M]
//
// (causal: -inf where d > 0).  Backward: dw[r, h] = sum of g[h, i, j] over row r.
// A head's matrix is constant along its diagonals j - i, so a tile of it is one
// window of values, and its gradient is a window of sums.
//
// Bound by memory: forward one write, backward one read.

#include <algorithm>

#include "ple_internal.h"
#include "ple_rows.h"

namespace ple {
namespace {

struct BiasArgs {
    const void *weight, *grad;
    const int32_t *buckets;      // [2 far + 1]
    const int64_t *starts;       // [B] or NULL: offset
    void *out;                   // forward: out; backward: the table's gradient
    float *partial;              // backward: [head, parts, stride]
    int64_t q, k, offset, tiles;
    int64_t rowblocks, colblocks;
    int B, H, R, far, causal;
    int rows, cols;              // of a tile
    int stride;                  // floats of a partial
    int weight_dtype;
};

// The position of a sample's first query (within what differences of 64 bits hold).
__device__ __forceinline__ int64_t start_of(const BiasArgs &a, int64_t b) {
    constexpr int64_t kMost = int64_t{1} << 60;
    return a.starts ? min(max(a.starts[b], -kMost), kMost) : a.offset;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------

constexpr int kBiasRows = 64, kBiasCols = 1024;      // a forward tile

// Elements of a type in 16 bytes, and how they lie in a dword.
template <int T>
constexpr int vec_elems() { return T == PLE_DTYPE_F32 ? 4 : 8; }

template <int T>
__device__ __forceinline__ uint32_t elem_bits(float v) {
    if constexpr (T == PLE_DTYPE_F32) return __float_as_uint(v);
    else return T == PLE_DTYPE_BF16 ? bf16_bits(v) : f16_bits(v);
}

// The value of a distance: the table's, 0 without a row, NaN beyond the table,
// -inf in a masked future.
__device__ __forceinline__ float bias_value(const BiasArgs &a, int h, int64_t d) {
    if (a.causal && d > 0) return -__builtin_inff();
    const int64_t c = min(max(d, static_cast<int64_t>(-a.far)), static_cast<int64_t>(a.far));
    const int r = a.buckets[c + a.far];
    if (r < 0) return 0.0f;
    if (r >= a.R) return __builtin_nanf("");
    return load_any(a.weight, static_cast<int64_t>(r) * a.H + h, a.weight_dtype);
}

// A tile's window of values lies in LDS once for every shift of less than a vector,
// so that a vector at any distance is one aligned read.
template <int T>
__global__ __launch_bounds__(kBlock) void ple_bias_forward_kernel(BiasArgs a) {
    constexpr int E = vec_elems<T>(), kBytes = elem_bytes(T);
    constexpr int kVecs = (kBiasCols + kBiasRows + E) / E + 1;       // of a shift's copy
    __shared__ uint4 s_copy[E][kVecs + 1];
    for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        int64_t t = tile;
        const int64_t c0 = t % a.colblocks * a.cols;
        t /= a.colblocks;
        const int64_t i0 = t % a.rowblocks * a.rows;
        const int64_t z = t / a.rowblocks;
        const int h = static_cast<int>(z % a.H);
        const int64_t start = start_of(a, z / a.H);
        const int64_t c1 = min(a.k, c0 + a.cols), i1 = min(a.q, i0 + a.rows);
        // the window: distances from `low` on
        const int64_t low = c0 - (start + i1 - 1);
        const int window = static_cast<int>(c1 - c0 + i1 - i0 - 1) + E;
        const int vecs = (window + E - 1) / E;
        __syncthreads();
        for (int i = threadIdx.x; i < (vecs + 1) * E; i += kBlock) {
            const uint32_t bits = elem_bits<T>(bias_value(a, h, low + i));
            if constexpr (T == PLE_DTYPE_F32) reinterpret_cast<uint32_t *>(s_copy[0])[i] = bits;
            else reinterpret_cast<uint16_t *>(s_copy[0])[i] = static_cast<uint16_t>(bits);
        }
        __syncthreads();
        for (int m = threadIdx.x; m < vecs; m += kBlock) {
            const uint4 u = s_copy[0][m], v = s_copy[0][m + 1];
            const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
            for (int s = 1; s < E; ++s) {
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (T == PLE_DTYPE_F32) o[j] = w[j + s];
                    else o[j] = s % 2 ? __builtin_amdgcn_alignbyte(w[j + s / 2 + 1], w[j + s / 2], 2) : w[j + s / 2];
                }
                s_copy[s][m] = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
        __syncthreads();
        // rows by waves: vectors at their 16-byte boundaries that begin in the tile, and
        // the elements before a row's first and after its last
        const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
        char *const out = static_cast<char *>(a.out);
        const uint64_t base = reinterpret_cast<uint64_t>(out) / kBytes;
        for (int64_t i = i0 + wave; i < i1; i += kWavesPerBlock) {
            const int64_t row = (z * a.q + i) * a.k;
            const int64_t at = c0 - (start + i) - low;            // window place of column c0
            const int skip = static_cast<int>((E - (base + row + c0) % E) % E);
            for (int64_t j = c0 + skip + lane * E; j < c1; j += kWave * E) {
                const int o = static_cast<int>(at + (j - c0));
                if (j + E <= a.k) {
                    *reinterpret_cast<uint4 *>(out + (row + j) * kBytes) = s_copy[o % E][o / E];
                } else {
                    for (int e = 0; e < a.k - j; ++e) {
                        if constexpr (T == PLE_DTYPE_F32)
                            reinterpret_cast<uint32_t *>(out)[row + j + e] = reinterpret_cast<const uint32_t *>(s_copy[0])[o + e];
                        else
                            reinterpret_cast<uint16_t *>(out)[row + j + e] = reinterpret_cast<const uint16_t *>(s_copy[0])[o + e];
                    }
                }
            }
            if (c0 == 0 && lane < skip && lane < a.k) {
                const int o = static_cast<int>(at) + lane;
                if constexpr (T == PLE_DTYPE_F32)
                    reinterpret_cast<uint32_t *>(out)[row + lane] = reinterpret_cast<const uint32_t *>(s_copy[0])[o];
                else
                    reinterpret_cast<uint16_t *>(out)[row + lane] = reinterpret_cast<const uint16_t *>(s_copy[0])[o];
            }
        }
    }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

constexpr int kGradRows = 64, kGradCols = 2048;      // a backward tile

// A tile's distances, and the places of a partial that they reach: lo to hi, with
// what lies beyond -far or far in the outermost.
struct Window {
    int64_t low;                 // distance of the window's first place
    int size;
    int64_t lo, hi;
    __device__ __forceinline__ Window(const BiasArgs &a, int64_t start, int64_t i0, int64_t c0) {
        const int64_t i1 = min(a.q, i0 + a.rows), c1 = min(a.k, c0 + a.cols);
        low = c0 - (start + i1 - 1);
        size = static_cast<int>(c1 - c0 + i1 - i0 - 1);
        const int64_t f = a.far;
        lo = min(max(low, -f), f);
        hi = min(max(low + size - 1, -f), f);
    }
};

__device__ __forceinline__ float sum_block(float v, float *lds) {
    v = group_sum<kWave>(v);
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kWavesPerBlock; ++i) s += lds[i];
    return s;
}

// Sums along a tile's diagonals.  Rows E apart (E: elements of 16 bytes) have their
// vector boundaries on the same diagonals, whatever the row's length; so a lane
// takes a vector of diagonals through every E-th row with aligned loads.
template <int T>
__global__ __launch_bounds__(kBlock) void ple_bias_backward_kernel(BiasArgs a) {
    constexpr int E = vec_elems<T>(), kBytes = elem_bytes(T), kSteps = kGradRows / E;
    constexpr int kPlaces = kGradCols + kGradRows + 2 * E;
    __shared__ float s_diag[kWavesPerBlock][kPlaces];
    __shared__ float s_sum[kWavesPerBlock];
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        int64_t t = tile;
        const int64_t c0 = t % a.colblocks * a.cols;
        t /= a.colblocks;
        const int64_t i0 = t % a.rowblocks * a.rows;
        const int64_t z = t / a.rowblocks;
        const int64_t start = start_of(a, z / a.H);
        const int64_t c1 = min(a.k, c0 + a.cols), i1 = min(a.q, i0 + a.rows);
        const Window win(a, start, i0, c0);
        // diagonal u = j - i; its distance is u - start
        const int64_t first = c0 - (i1 - 1), last = c1 - 1 - i0;
        __syncthreads();
        for (int i = threadIdx.x; i < kWavesPerBlock * kPlaces; i += kBlock) s_diag[0][i] = 0.0f;
        __syncthreads();
        const char *const grad = static_cast<const char *>(a.grad) + z * a.q * a.k * kBytes;
        const uint64_t base = reinterpret_cast<uint64_t>(grad) / kBytes;
        for (int c = wave; c < E && i0 + c < i1; c += kWavesPerBlock) {
            const int64_t i = i0 + c;
            // the first diagonal at or before `first` whose vectors are aligned in these rows
            const int64_t back = static_cast<int64_t>((base + i * (a.k + 1) + first) & (E - 1));
            for (int64_t u = first - back + lane * E; u <= last; u += kWave * E) {
                if (a.causal && u > start) break;
                float acc[E] = {};
#pragma unroll
                for (int s = 0; s < kSteps; ++s) {
                    const int64_t r = i + s * E, j = u + r;
                    if (r >= i1 || j >= c1 || j + E <= c0) continue;
                    const char *const p = grad + (r * a.k + j) * kBytes;
                    float v[E];
                    if (j >= c0 && j + E <= c1) {
                        load_vec<T, E>(p, 0, v);
                    } else {
#pragma unroll
                        for (int e = 0; e < E; ++e) v[e] = j + e >= c0 && j + e < c1 ? load_grad<T>(p, e) : 0.0f;
                    }
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e] += v[e];
                }
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int at = static_cast<int>(u + e - first) + E;
                    s_diag[wave][at] += acc[e];
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
        __syncthreads();
        const int64_t parts = a.B * a.rowblocks * a.colblocks;
        const int64_t part = ((z / a.H) * a.rowblocks + i0 / a.rows) * a.colblocks + c0 / a.cols;
        float *const partial = a.partial + ((z % a.H) * parts + part) * a.stride;
        float before = 0.0f, after = 0.0f;
        for (int w = threadIdx.x; w < win.size; w += kBlock) {
            const int64_t d = win.low + w;
            if (a.causal && d > 0) break;
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < kWavesPerBlock; ++v) s += s_diag[v][w + E];
            if (d <= win.lo) before += s;
            else if (d >= win.hi) after += s;
            else partial[d - win.lo] = s;
        }
        before = sum_block(before, s_sum);
        after = sum_block(after, s_sum);
        if (threadIdx.x == 0) {
            partial[0] = win.hi > win.lo ? before : before + after;
            if (win.hi > win.lo) partial[win.hi - win.lo] = after;
        }
        // (masked distances between lo and hi have nothing)
        if (a.causal)
            for (int64_t e = max(win.lo + 1, static_cast<int64_t>(1)) + threadIdx.x; e < win.hi; e += kBlock) partial[e - win.lo] = 0.0f;
    }
}

// Sums of a head's distances over the tiles, then of each row's distances: a wave a
// row.  Workgroups take a head and kJoinRows rows of the table.
constexpr int kJoinRows = 64, kJoinPlaces = 4096, kJoinThreads = 1024;

__global__ __launch_bounds__(kJoinThreads) void ple_bias_join_kernel(BiasArgs a) {
    __shared__ float s_sum[kJoinPlaces];
    __shared__ float s_row[kJoinRows];
    const int64_t groups = (a.R + kJoinRows - 1) / kJoinRows;
    const int64_t parts = a.B * a.rowblocks * a.colblocks;
    const int64_t places = 2 * static_cast<int64_t>(a.far) + 1;
    for (int64_t unit = blockIdx.x; unit < a.H * groups; unit += gridDim.x) {
        const int h = static_cast<int>(unit / groups);
        const int r0 = static_cast<int>(unit % groups) * kJoinRows, rows = min(kJoinRows, a.R - r0);
        __syncthreads();
        if (threadIdx.x < kJoinRows) s_row[threadIdx.x] = 0.0f;
        for (int64_t p0 = 0; p0 < places; p0 += kJoinPlaces) {
            const int count = static_cast<int>(min(places - p0, static_cast<int64_t>(kJoinPlaces)));
            __syncthreads();
            for (int i = threadIdx.x; i < count; i += kJoinThreads) {
                const int64_t e = p0 + i - a.far;
                float s = 0.0f;
                for (int64_t b = 0; b < a.B; ++b) {
                    const int64_t start = start_of(a, b);
                    for (int64_t y = 0; y < a.rowblocks; ++y)
                        for (int64_t x = 0; x < a.colblocks; ++x) {
                            const Window win(a, start, y * a.rows, x * a.cols);
                            if (e < win.lo || e > win.hi) continue;
                            s += a.partial[(h * parts + (b * a.rowblocks + y) * a.colblocks + x) * a.stride + (e - win.lo)];
                        }
                }
                s_sum[i] = s;
            }
            __syncthreads();
            for (int r = threadIdx.x / kWave; r < rows; r += kJoinThreads / kWave) {
                float s = 0.0f;
                for (int i = threadIdx.x % kWave; i < count; i += kWave)
                    if (a.buckets[p0 + i] == r0 + r) s += s_sum[i];
                s = group_sum<kWave>(s);
                if (threadIdx.x % kWave == 0) s_row[r] += s;
            }
        }
        __syncthreads();
        if (threadIdx.x < rows) store_any(a.out, static_cast<int64_t>(r0 + threadIdx.x) * a.H + h, s_row[threadIdx.x], a.weight_dtype);
    }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

constexpr int64_t kMaxGrid = 1 << 20;

BiasArgs bias_args(const BiasRequest &r, int rows, int cols) {
    BiasArgs a{};
    a.weight = r.weight; a.grad = r.grad; a.buckets = r.buckets; a.starts = r.starts;
    a.partial = static_cast<float *>(r.workspace);
    a.q = r.q; a.k = r.k; a.offset = r.offset;
    a.B = static_cast<int>(r.B); a.H = static_cast<int>(r.H); a.R = static_cast<int>(r.R); a.far = static_cast<int>(r.far);
    a.causal = r.causal;
    a.rows = rows; a.cols = cols;
    a.rowblocks = (r.q + rows - 1) / rows;
    a.colblocks = (r.k + cols - 1) / cols;
    a.tiles = r.B * r.H * a.rowblocks * a.colblocks;
    a.stride = static_cast<int>(std::min<int64_t>(std::min<int64_t>(rows, r.q) + std::min<int64_t>(cols, r.k) - 1, 2 * r.far + 1));
    a.weight_dtype = r.weight_dtype;
    return a;
}

template <typename F>
hipError_t with_type(int dtype, F f) {
    if (dtype == PLE_DTYPE_F32) return f(std::integral_constant<int, PLE_DTYPE_F32>{});
    if (dtype == PLE_DTYPE_F16) return f(std::integral_constant<int, PLE_DTYPE_F16>{});
    return f(std::integral_constant<int, PLE_DTYPE_BF16>{});
}

}  // namespace

int bias_run(const BiasRequest &r) {
    BiasArgs a = bias_args(r, kBiasRows, kBiasCols);
    a.out = r.out;
    const dim3 grid(static_cast<unsigned>(std::min(a.tiles, kMaxGrid)));
    return static_cast<int>(with_type(r.out_dtype, [&](auto t) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_bias_forward_kernel<decltype(t)::value>), grid, dim3(kBlock), 0, r.stream, a);
        return hipGetLastError();
    }));
}

size_t bias_backward_workspace_bytes(const BiasRequest &r) {
    const BiasArgs a = bias_args(r, kGradRows, kGradCols);
    return align_up(static_cast<size_t>(a.tiles) * a.stride * 4, 256);
}

int bias_backward_run(const BiasRequest &r) {
    const size_t need = bias_backward_workspace_bytes(r);
    if (need > 0 && (!r.workspace || r.workspace_bytes < need || reinterpret_cast<uintptr_t>(r.workspace) % 256 != 0))
        return PLE_E_WORKSPACE;
    BiasArgs a = bias_args(r, kGradRows, kGradCols);
    a.out = r.dw;
    if (a.tiles > 0) {
        const dim3 grid(static_cast<unsigned>(std::min(a.tiles, kMaxGrid)));
        const hipError_t rc = with_type(r.out_dtype, [&](auto t) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_bias_backward_kernel<decltype(t)::value>), grid, dim3(kBlock), 0, r.stream, a);
            return hipGetLastError();
        });
        if (rc != hipSuccess) return static_cast<int>(rc);
    }
    const int64_t units = r.H * ((r.R + kJoinRows - 1) / kJoinRows);
    hipLaunchKernelGGL(ple_bias_join_kernel, dim3(static_cast<unsigned>(std::min(units, kMaxGrid))), dim3(kJoinThreads), 0, r.stream, a);
    return static_cast<int>(hipGetLastError());
}

}  // namespace ple

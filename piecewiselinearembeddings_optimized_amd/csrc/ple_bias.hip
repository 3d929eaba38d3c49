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
// Bound by memory: forward one write, backward one read.  Measured: 16 x 2048 x 2048
// bf16 25 us (5.3 TB/s) and 29 us (4.6 TB/s) with 11 us of joins; 16 x 4096 x 4096 108 us
// and 67 us (causal: half of it is read) with 20 us; one query, 64 x 32 x 1 x 4097, 10 us.

#include <algorithm>
#include <type_traits>

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
    float *total;                // backward: [head, 2 far + 1] sums of the parts, or NULL
    int64_t q, k, offset, tiles;
    int64_t rowblocks, colblocks;
    int B, H, R, far, causal;
    int heads, headblocks;       // few queries: heads of a tile
    int rows, cols;              // forward: of a tile; backward: diagonals of a unit ...
    int reach;                   // ... and before them
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

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// NT: past the caches
template <bool NT>
__device__ __forceinline__ void store16(char *p, const uint4 &w) {
    const u32x4 v = {w.x, w.y, w.z, w.w};
    if constexpr (NT) __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(p));
    else *reinterpret_cast<u32x4 *>(p) = v;
}

template <int T>
__device__ __forceinline__ void store_bits(char *out, int64_t i, uint32_t bits) {
    if constexpr (T == PLE_DTYPE_F32) reinterpret_cast<uint32_t *>(out)[i] = bits;
    else reinterpret_cast<uint16_t *>(out)[i] = static_cast<uint16_t>(bits);
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
template <int T, bool NT>
__global__ __launch_bounds__(kBlock) void ple_bias_forward_kernel(BiasArgs a) {
    constexpr int E = vec_elems<T>(), kBytes = elem_bytes(T);
    constexpr int kVecs = (kBiasCols + kBiasRows + E) / E + 2;       // of a shift's copy
    __shared__ uint4 s_copy[E * kVecs];
    char *const s_elem = reinterpret_cast<char *>(s_copy);           // the copy without a shift
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
        for (int i = threadIdx.x; i < (vecs + 1) * E; i += kBlock) store_bits<T>(s_elem, i, elem_bits<T>(bias_value(a, h, low + i)));
        __syncthreads();
        for (int m = threadIdx.x; m < vecs; m += kBlock) {
            const uint4 u = s_copy[m], v = s_copy[m + 1];
            const uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
            for (int s = 1; s < E; ++s) {
                uint32_t o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (T == PLE_DTYPE_F32) o[j] = w[j + s];
                    else o[j] = s % 2 ? __builtin_amdgcn_alignbyte(w[j + s / 2 + 1], w[j + s / 2], 2) : w[j + s / 2];
                }
                s_copy[s * kVecs + m] = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
        __syncthreads();
        // rows by waves: vectors at their 16-byte boundaries that begin in the tile, and
        // the elements before a row's first and after its last
        const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
        char *const out = static_cast<char *>(a.out);
        const uint64_t base = reinterpret_cast<uint64_t>(out) / kBytes;
        const auto one = [&](int o) {
            if constexpr (T == PLE_DTYPE_F32) return reinterpret_cast<const uint32_t *>(s_elem)[o];
            else return static_cast<uint32_t>(reinterpret_cast<const uint16_t *>(s_elem)[o]);
        };
        for (int64_t i = i0 + wave; i < i1; i += kWavesPerBlock) {
            const int64_t row = (z * a.q + i) * a.k;
            const int at = static_cast<int>(c0 - (start + i) - low);            // window place of column c0
            const int skip = static_cast<int>((E - (base + row + c0) % E) % E);
            for (int64_t j = c0 + skip + lane * E; j < c1; j += kWave * E) {
                const int o = at + static_cast<int>(j - c0);
                if (j + E <= a.k)
                    store16<NT>(out + (row + j) * kBytes, s_copy[o % E * kVecs + o / E]);
                else
                    for (int e = 0; e < a.k - j; ++e) store_bits<T>(out, row + j + e, one(o + e));
            }
            if (c0 == 0 && lane < skip && lane < a.k) store_bits<T>(out, row + lane, one(at + lane));
        }
    }
}

// Few queries (a generated token): a row has no other rows to share a window with, but
// its heads share its buckets.  A workgroup takes kFewCols columns of a row: their
// table rows in LDS, once for every shift; then its heads, each value looked up there.
// (The heads' tables take the LDS that they need: with room for the largest, four
// workgroups a CU, 64 x 32 x 1 x 4096 fp32 took 12.6 us, so 10.2.)
constexpr int kFewCols = 1024, kFewTable = 8192;     // columns; values of the heads' tables

template <int T>
__global__ __launch_bounds__(kBlock) void ple_bias_few_kernel(BiasArgs a) {
    constexpr int E = vec_elems<T>(), kBytes = elem_bytes(T);
    constexpr int kVecs = kFewCols / E + 3;
    using Bits = std::conditional_t<T == PLE_DTYPE_F32, uint32_t, uint16_t>;
    struct alignas(2 * E) Slots { uint16_t r[E]; };
    __shared__ Slots s_slot[E * kVecs];
    extern __shared__ uint32_t s_tables[];               // the heads' tables
    Bits *const s_table = reinterpret_cast<Bits *>(s_tables);
    uint16_t *const s_each = reinterpret_cast<uint16_t *>(s_slot);
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    // places of a head's table: the rows, then 0 (no row), NaN (beyond the table), -inf (masked)
    const int places = a.R + 3;
    for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        int64_t t = tile;
        const int64_t c0 = t % a.colblocks * a.cols;
        t /= a.colblocks;
        const int h0 = static_cast<int>(t % a.headblocks) * a.heads, h1 = min(a.H, h0 + a.heads);
        t /= a.headblocks;
        const int64_t i = t % a.q, b = t / a.q;
        const int64_t position = start_of(a, b) + i, c1 = min(a.k, c0 + a.cols);
        __syncthreads();
        for (int p = threadIdx.x; p < (h1 - h0) * places; p += kBlock) {
            const int h = p / places, r = p - h * places;
            float v = r == a.R ? 0.0f : r == a.R + 1 ? __builtin_nanf("") : -__builtin_inff();
            if (r < a.R) v = load_any(a.weight, static_cast<int64_t>(r) * a.H + h0 + h, a.weight_dtype);
            s_table[p] = static_cast<Bits>(elem_bits<T>(v));
        }
        const int vecs = static_cast<int>(c1 - c0 + E - 1) / E + 1;
        for (int c = threadIdx.x; c < (vecs + 1) * E; c += kBlock) {
            const int64_t d = c0 + c - position;
            int r = a.R + 2;
            if (!(a.causal && d > 0)) {
                const int64_t f = a.far;
                r = a.buckets[min(max(d, -f), f) + f];
                r = r < 0 ? a.R : r >= a.R ? a.R + 1 : r;
            }
            s_each[c] = static_cast<uint16_t>(r);
        }
        __syncthreads();
        for (int m = threadIdx.x; m < vecs; m += kBlock) {
            uint32_t w[E];           // two vectors of slots
            __builtin_memcpy(w, &s_slot[m], 2 * sizeof(Slots));
#pragma unroll
            for (int s = 1; s < E; ++s) {
                uint32_t o[E / 2];
#pragma unroll
                for (int j = 0; j < E / 2; ++j)
                    o[j] = s % 2 ? __builtin_amdgcn_alignbyte(w[j + s / 2 + 1], w[j + s / 2], 2) : w[j + s / 2];
                __builtin_memcpy(&s_slot[s * kVecs + m], o, sizeof(Slots));
            }
        }
        __syncthreads();
        char *const out = static_cast<char *>(a.out);
        const uint64_t base = reinterpret_cast<uint64_t>(out) / kBytes;
        for (int h = h0 + wave; h < h1; h += kWavesPerBlock) {
            const Bits *const table = s_table + (h - h0) * places;
            const int64_t row = ((b * a.H + h) * a.q + i) * a.k;
            const int skip = static_cast<int>((E - (base + row + c0) % E) % E);
            for (int64_t j = c0 + skip + lane * E; j < c1; j += kWave * E) {
                const int o = static_cast<int>(j - c0);
                const Slots slots = s_slot[skip * kVecs + o / E];
                uint32_t w[4];
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    if constexpr (T == PLE_DTYPE_F32) w[p] = table[slots.r[p]];
                    else w[p] = table[slots.r[2 * p]] | static_cast<uint32_t>(table[slots.r[2 * p + 1]]) << 16;
                }
                if (j + E <= a.k)
                    store16<false>(out + (row + j) * kBytes, make_uint4(w[0], w[1], w[2], w[3]));
                else
                    for (int e = 0; e < a.k - j; ++e) store_bits<T>(out, row + j + e, table[s_each[o + e]]);
            }
            if (c0 == 0 && lane < skip && lane < a.k) store_bits<T>(out, row + lane, table[s_each[lane]]);
        }
    }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------

constexpr int kGradRows = 64;            // rows of a wave's unit
constexpr int kGradItems = 8;            // in so many steps of
constexpr int kGradLoads = 8;            // loads a lane

// A wave's unit: kGradRows rows of a sample's head along 64 vectors of diagonals j - i
// (a parallelogram of the matrix, so no unit has edges inside it), and the places of
// its partial: distances lo to hi, with what lies beyond -far or far in the outermost.
// Vectors begin up to reach diagonals before `first`, as the rows' addresses have it.
// live: whether any distance counts.
struct Unit {
    int64_t first;               // diagonal
    int64_t low;                 // distance of the first place, first - reach
    int size;
    int64_t lo, hi;
    bool live;
    __device__ __forceinline__ Unit(const BiasArgs &a, int64_t start, int64_t i0, int64_t chunk) {
        const int64_t i1 = min(a.q, i0 + kGradRows);
        first = chunk * a.cols - (i1 - 1);
        low = first - a.reach - start;
        size = a.cols + a.reach;
        const int64_t f = a.far, top = a.causal ? 0 : f;
        live = low <= top || !a.causal;
        lo = min(max(low, -f), top);
        hi = min(max(low + size - 1, -f), top);
    }
};

// Elements of a vector as loaded.
template <int T>
__device__ __forceinline__ float vector_elem(const uint4 &raw, int e) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    return grad_elem<T>(w, e);
}

// A vector without its elements before column 0 and from column k on; j: its first
// element's column.
template <int T>
__device__ __forceinline__ uint4 within(const uint4 &raw, int64_t j, int64_t k) {
    uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (T == PLE_DTYPE_F32) {
            w[i] = j + i >= 0 && j + i < k ? w[i] : 0u;
        } else {
            const uint32_t lo = j + 2 * i >= 0 && j + 2 * i < k ? 0xffffu : 0u;
            const uint32_t hi = j + 2 * i + 1 >= 0 && j + 2 * i + 1 < k ? 0xffff0000u : 0u;
            w[i] &= lo | hi;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Adds vectors that begin BACK diagonals before the lane's own to its sums
// (sum[E - 1 + x]: x diagonals after its own first).
template <int T, int BACK, int N>
__device__ __forceinline__ void add_vectors(const uint4 (&raw)[N], float (&sum)[2 * vec_elems<T>() - 1]) {
    constexpr int E = vec_elems<T>();
#pragma unroll
    for (int v = 0; v < N; ++v)
#pragma unroll
        for (int e = 0; e < E; ++e) sum[E - 1 - BACK + e] += vector_elem<T>(raw[v], e);
}

template <int T, int N>
__device__ __forceinline__ void add_vectors(const uint4 (&raw)[N], int back, float (&sum)[2 * vec_elems<T>() - 1]) {
    switch (back) {
        case 0: return add_vectors<T, 0>(raw, sum);
        case 1: return add_vectors<T, 1>(raw, sum);
        case 2: return add_vectors<T, 2>(raw, sum);
        case 3: return add_vectors<T, 3>(raw, sum);
        default: break;
    }
    if constexpr (vec_elems<T>() == 8) {
        switch (back) {
            case 4: return add_vectors<T, 4>(raw, sum);
            case 5: return add_vectors<T, 5>(raw, sum);
            case 6: return add_vectors<T, 6>(raw, sum);
            default: return add_vectors<T, 7>(raw, sum);
        }
    }
}

// Elements of the gradient (samples times heads alone may pass 32 bits).
__device__ __forceinline__ int64_t elements(const BiasArgs &a) { return static_cast<int64_t>(a.B) * a.H * a.q * a.k; }

// The tensor's first elements that lie before its first 16-byte boundary, and its last
// ones behind the last: the vectors that hold them are not all in its memory.
// (apart_last of them end the last row, which has all of them: k >= E)
template <int T>
__device__ __forceinline__ int apart_first(const BiasArgs &a) {
    constexpr int E = vec_elems<T>();
    return (E - static_cast<int>(reinterpret_cast<uint64_t>(a.grad) / elem_bytes(T) % E)) % E;
}

template <int T>
__device__ __forceinline__ int apart_last(const BiasArgs &a) {
    constexpr int E = vec_elems<T>();
    return static_cast<int>((reinterpret_cast<uint64_t>(a.grad) / elem_bytes(T) + elements(a)) % E);
}

// Sums along diagonals.  Rows E apart (E: elements of 16 bytes) have their vector
// boundaries on the same diagonals, whatever the row's length; so a lane takes a vector
// of diagonals through every E-th row with aligned loads, and the next rows with
// another shift.  NARROW: rows of less than a vector, element by element.
template <int T, bool NARROW>
__global__ __launch_bounds__(kBlock, 4) void ple_bias_backward_kernel(BiasArgs a) {
    constexpr int E = vec_elems<T>(), kBytes = elem_bytes(T);
    constexpr int kEach = kGradItems / E;                    // steps of a class of rows
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int64_t parts = a.B * a.rowblocks * a.colblocks;
    for (int64_t unit = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + wave; unit < a.tiles;
         unit += static_cast<int64_t>(gridDim.x) * kWavesPerBlock) {
        const int64_t t = unit / a.colblocks, chunk = unit - t * a.colblocks;
        const int64_t z = t / a.rowblocks, block = t - z * a.rowblocks, i0 = block * kGradRows;
        const int64_t b = z / a.H, start = start_of(a, b);
        const Unit win(a, start, i0, chunk);
        if (!win.live) continue;
        const int rows = static_cast<int>(min(a.q - i0, static_cast<int64_t>(kGradRows)));
        const char *const row0 = static_cast<const char *>(a.grad) + (z * a.q + i0) * a.k * kBytes;
        const int64_t own = win.first + lane * E;            // the lane's first diagonal
        const int64_t col = own + i0;                        // ... its column in row i0
        float mine[E], before_own[E - 1];
        if constexpr (NARROW) {
#pragma unroll
            for (int d = 0; d < E; ++d) {
                mine[d] = 0.0f;
                if (d < E - 1) before_own[d] = 0.0f;
                for (int j = 0; j < a.k; ++j) {
                    const int64_t r = j - (col + d);
                    if (r >= 0 && r < rows) mine[d] += load_grad<T>(row0, r * a.k + j);
                }
            }
        } else {
            const int64_t step = (a.k + 1) * kBytes;         // from row to row
            const uint64_t place = reinterpret_cast<uint64_t>(row0) / kBytes + static_cast<uint64_t>(col);
            const bool dead = a.causal && own - (E - 1) > start;
            // vectors that leave the tensor are read by the join
            const int skip_first = z == 0 && i0 == 0 ? 0 : -1;
            const int skip_last = z + 1 == static_cast<int64_t>(a.B) * a.H && i0 + rows == a.q ? rows - 1 : -1;
            // The lane's part of an address is the same in every row, the rows' is scalar;
            // lanes outside of a row get zeros.
            const __amdgpu_buffer_rsrc_t rs = make_rsrc(row0 + (win.first + i0 - (E - 1)) * kBytes, 0xfffffff0u);
            const uint32_t at = static_cast<uint32_t>(lane) * 16;
            float sum[2 * E - 1] = {};
#pragma unroll 1
            for (int item = 0; item < kGradItems; ++item) {
                // the item's first row, and how far before the lane's diagonal its vectors begin
                const int c = item / kEach + item % kEach * kGradLoads * E;
                const int back = __builtin_amdgcn_readfirstlane(
                    static_cast<int>(place + static_cast<uint64_t>(c) * static_cast<uint64_t>(a.k + 1)) & (E - 1));
                if (c >= rows) continue;
                const uint32_t from = static_cast<uint32_t>((E - 1 - back) * kBytes) + static_cast<uint32_t>(c * step);
                // (columns E - 1 further than they are, so that all of a row's are positive)
                const uint32_t j = static_cast<uint32_t>(col - back + c + (E - 1)), k = static_cast<uint32_t>(a.k + (E - 1));
                uint4 raw[kGradLoads];
                bool cut = false;
#pragma unroll
                for (int v = 0; v < kGradLoads; ++v) {
                    const int r = c + v * E;
                    const uint32_t jv = j + v * E;
                    const bool part = jv < E - 1 || jv + E > k;
                    const bool on = jv < k && r < rows && !dead &&
                                    !(r == skip_first && jv < E - 1) && !(r == skip_last && jv + E > k);
                    const auto w = __builtin_amdgcn_raw_buffer_load_b128(
                        rs, on ? at : 0xffffffffu, __builtin_amdgcn_readfirstlane(from + static_cast<uint32_t>(v * E * step)), 0);
                    raw[v] = make_uint4(w[0], w[1], w[2], w[3]);
                    cut = cut || (on && part);
                }
                if (__any(cut)) {
#pragma unroll
                    for (int v = 0; v < kGradLoads; ++v) raw[v] = within<T>(raw[v], col - back + c + v * E, a.k);
                }
                add_vectors<T>(raw, back, sum);
            }
            // the lane's own diagonals: with what the next lane's vectors have of them
            mine[0] = sum[E - 1];
#pragma unroll
            for (int d = 0; d < E - 1; ++d) {
                before_own[d] = sum[d];
                const float next = __shfl_down(sum[d], 1);
                mine[d + 1] = sum[E + d] + (lane < kWave - 1 ? next : 0.0f);
            }
        }
        float *const partial = a.partial + ((z - b * a.H) * parts + (b * a.rowblocks + block) * a.colblocks + chunk) * a.stride;
        float before = 0.0f, after = 0.0f;
        const auto leave = [&](int64_t d, float s) {
            if (a.causal && d > 0) return;
            if (d <= win.lo) before += s;
            else if (d >= win.hi) after += s;
            else partial[d - win.lo] = s;
        };
#pragma unroll
        for (int d = 0; d < E; ++d) leave(own + d - start, mine[d]);
        if (lane == 0)
#pragma unroll
            for (int d = 0; d < E - 1; ++d) leave(win.low + d, before_own[d]);
        before = group_sum<kWave>(before);
        after = group_sum<kWave>(after);
        if (lane == 0) {
            partial[0] = win.hi > win.lo ? before : before + after;
            if (win.hi > win.lo) partial[win.hi - win.lo] = after;
        }
    }
}

// What of a head's sum at distance e lies in vectors that leave the tensor.
template <int T>
__device__ __forceinline__ float apart_sum(const BiasArgs &a, int h, int e) {
    float s = 0.0f;
    if (a.k < vec_elems<T>()) return s;
    const int first = apart_first<T>(a), last = apart_last<T>(a);
    const int64_t far = a.far, end = elements(a);
    const auto add = [&](int64_t at, int64_t b, int64_t i, int64_t j) {
        const int64_t d = j - start_of(a, b) - i;
        if (!(a.causal && d > 0) && min(max(d, -far), far) == e) s += load_grad<T>(a.grad, at);
    };
    if (h == 0)
        for (int j = 0; j < first; ++j) add(j, 0, 0, j);
    if (h == a.H - 1)
        for (int64_t j = a.k - last; j < a.k; ++j)
            if (end - a.k + j >= first) add(end - a.k + j, a.B - 1, a.q - 1, j);
    return s;
}

// Sums of a head's distances over the units: 64 distances a workgroup.  It lists the
// units that reach them, and its waves take one of these each in turn.
constexpr int kJoinThreads = 1024;

template <int T>
__global__ __launch_bounds__(kJoinThreads) void ple_bias_total_kernel(BiasArgs a) {
    __shared__ float s_sum[kJoinThreads];
    __shared__ int64_t s_base[kJoinThreads];             // a unit's place of distance 0
    __shared__ int s_lo[kJoinThreads], s_hi[kJoinThreads];
    __shared__ int s_count[kJoinThreads / kWave];
    const int64_t places = 2 * static_cast<int64_t>(a.far) + 1, blocks = (places + kWave - 1) / kWave;
    const int64_t parts = a.B * a.rowblocks * a.colblocks;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    for (int64_t unit = blockIdx.x; unit < a.H * blocks; unit += gridDim.x) {
        const int h = static_cast<int>(unit / blocks);
        const int64_t place = (unit - h * blocks) * kWave + lane;
        const int e = static_cast<int>(place - a.far), e0 = e - lane;
        const float *const head = a.partial + h * parts * a.stride;
        // sums of units whose distances are all -far or less (fold[0]), or the most that
        // counts and more: a thread a unit
        const int top = a.causal ? 0 : a.far;
        float s = 0.0f, fold[2] = {};
        for (int64_t p0 = 0; p0 < parts && e0 <= top; p0 += kJoinThreads) {
            const int64_t part = p0 + threadIdx.x;
            bool hit = false;
            int lo = 0, hi = 0;
            if (part < parts) {
                const int64_t by = part / a.colblocks, b = by / a.rowblocks;
                const Unit win(a, start_of(a, b), (by - b * a.rowblocks) * kGradRows, part - by * a.colblocks);
                lo = static_cast<int>(win.lo);
                hi = static_cast<int>(win.hi);
                hit = win.live && lo < e0 + kWave && hi >= e0;
                if (hit && lo == hi) {
                    fold[lo == top] += head[part * a.stride];
                    hit = false;
                }
            }
            const uint64_t hits = __ballot(hit);
            __syncthreads();
            if (lane == 0) s_count[wave] = __popcll(hits);
            __syncthreads();
            int at = __popcll(hits & ((uint64_t{1} << lane) - 1)), count = 0;
#pragma unroll
            for (int w = 0; w < kJoinThreads / kWave; ++w) {
                if (w < wave) at += s_count[w];
                count += s_count[w];
            }
            if (hit) {
                s_base[at] = part * a.stride - lo;
                s_lo[at] = lo;
                s_hi[at] = hi;
            }
            __syncthreads();
#pragma unroll 4
            for (int i = wave; i < count; i += kJoinThreads / kWave)
                if (e >= s_lo[i] && e <= s_hi[i]) s += head[s_base[i] + e];
        }
        fold[0] = group_sum<kWave>(fold[0]);
        fold[1] = group_sum<kWave>(fold[1]);
        if (e == -a.far) s += fold[0];
        if (e == top) s += fold[1];
        __syncthreads();
        s_sum[threadIdx.x] = s;
        __syncthreads();
        if (wave == 0 && place < places) {
            for (int w = 1; w < kJoinThreads / kWave; ++w) s += s_sum[w * kWave + lane];
            if (parts > 0) s += apart_sum<T>(a, h, e);
            a.total[h * places + place] = s;
        }
    }
}

// Sums of each row's distances: a wave a row.  Workgroups take a head and kJoinRows
// rows of the table.
constexpr int kJoinRows = 16, kJoinPlaces = 4096;

__global__ __launch_bounds__(kJoinThreads) void ple_bias_join_kernel(BiasArgs a) {
    __shared__ float s_sum[kJoinPlaces];
    __shared__ int s_bucket[kJoinPlaces];
    __shared__ float s_row[kJoinRows];
    const int64_t groups = (a.R + kJoinRows - 1) / kJoinRows;
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
                s_sum[i] = a.total[h * places + p0 + i];
                s_bucket[i] = a.buckets[p0 + i];
            }
            __syncthreads();
            for (int r = threadIdx.x / kWave; r < rows; r += kJoinThreads / kWave) {
                float s = 0.0f;
#pragma unroll 4
                for (int i = threadIdx.x % kWave; i < count; i += kWave) s += s_bucket[i] == r0 + r ? s_sum[i] : 0.0f;
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

BiasArgs bias_args(const BiasRequest &r) {
    BiasArgs a{};
    a.weight = r.weight; a.grad = r.grad; a.buckets = r.buckets; a.starts = r.starts;
    a.partial = static_cast<float *>(r.workspace);
    a.q = r.q; a.k = r.k; a.offset = r.offset;
    a.B = static_cast<int>(r.B); a.H = static_cast<int>(r.H); a.R = static_cast<int>(r.R); a.far = static_cast<int>(r.far);
    a.causal = r.causal;
    a.weight_dtype = r.weight_dtype;
    return a;
}

// Columns in tiles of about one size, whole vectors of each type, at most `most`.
void split_columns(BiasArgs &a, int most) {
    a.colblocks = (a.k + most - 1) / most;
    a.cols = static_cast<int>(((a.k + a.colblocks - 1) / a.colblocks + 7) / 8 * 8);
}

// Tiles of fewer rows where there are not four for every CU.  (12 x 1023 x 1301 fp32: of
// 16 rows 14.8 us, of 64 17.3)
BiasArgs forward_args(const BiasRequest &r) {
    BiasArgs a = bias_args(r);
    a.out = r.out;
    split_columns(a, kBiasCols);
    for (a.rows = kBiasRows;; a.rows /= 2) {
        a.rowblocks = (r.q + a.rows - 1) / a.rows;
        a.tiles = r.B * r.H * a.rowblocks * a.colblocks;
        if (a.rows <= 8 || a.tiles >= 4 * device_cu_count()) return a;
    }
}

// Rows that have few others of their sample's head, and a table of which some heads fit.
bool few_rows(const BiasRequest &r) { return r.q < 8 && r.R + 3 <= kFewTable; }

BiasArgs few_args(const BiasRequest &r) {
    BiasArgs a = bias_args(r);
    a.out = r.out;
    split_columns(a, kFewCols);
    // heads of a tile: as many as fit, but as many tiles as run at once, four a CU
    const int64_t rows = r.B * r.q * a.colblocks, fit = std::min<int64_t>(r.H, kFewTable / (r.R + 3));
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(r.H, 4 * device_cu_count() / rows));
    a.heads = static_cast<int>(std::min(fit, (r.H + blocks - 1) / blocks));
    a.headblocks = static_cast<int>((r.H + a.heads - 1) / a.heads);
    a.tiles = rows * a.headblocks;
    return a;
}

// elems: elements of 16 bytes of the gradient
BiasArgs backward_args(const BiasRequest &r, int elems) {
    BiasArgs a = bias_args(r);
    a.out = r.dw;
    a.rows = kGradRows; a.cols = kWave * elems; a.reach = elems - 1;
    a.rowblocks = (r.q + kGradRows - 1) / kGradRows;
    // a block's diagonals, and what vectors that begin before them miss at the end
    a.colblocks = r.q > 0 && r.k > 0 ? (r.k + std::min<int64_t>(r.q, kGradRows) - 1 + a.reach + a.cols - 1) / a.cols : 0;
    a.tiles = r.B * r.H * a.rowblocks * a.colblocks;
    a.stride = static_cast<int>(std::min<int64_t>(a.cols + a.reach, 2 * r.far + 1));
    return a;
}

size_t partial_bytes(const BiasArgs &a) { return align_up(static_cast<size_t>(a.tiles) * a.stride * 4, 256); }

template <typename F>
hipError_t with_type(int dtype, F f) {
    if (dtype == PLE_DTYPE_F32) return f(std::integral_constant<int, PLE_DTYPE_F32>{});
    if (dtype == PLE_DTYPE_F16) return f(std::integral_constant<int, PLE_DTYPE_F16>{});
    return f(std::integral_constant<int, PLE_DTYPE_BF16>{});
}

}  // namespace

int bias_run(const BiasRequest &r) {
    if (few_rows(r)) {
        const BiasArgs a = few_args(r);
        return static_cast<int>(with_type(r.out_dtype, [&](auto t) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_bias_few_kernel<decltype(t)::value>),
                               dim3(static_cast<unsigned>(std::min(a.tiles, kMaxGrid))), dim3(kBlock),
                               static_cast<size_t>(a.heads) * (a.R + 3) * elem_bytes(decltype(t)::value), r.stream, a);
            return hipGetLastError();
        }));
    }
    const BiasArgs a = forward_args(r);
    const dim3 grid(static_cast<unsigned>(std::min(a.tiles, kMaxGrid)));
    // An output that the memory-side cache (256 MB) cannot hold goes past the caches, so
    // that what runs next does not wait for its writes (forward and backward of 537 MB
    // bf16 223 us with plain stores, 194 without; of 134 MB 64 with, 66 without).
    const bool stream = r.B * r.H * r.q * r.k * elem_bytes(r.out_dtype) > (int64_t{256} << 20);
    return static_cast<int>(with_type(r.out_dtype, [&](auto t) {
        constexpr int T = decltype(t)::value;
        if (stream) hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_bias_forward_kernel<T, true>), grid, dim3(kBlock), 0, r.stream, a);
        else hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_bias_forward_kernel<T, false>), grid, dim3(kBlock), 0, r.stream, a);
        return hipGetLastError();
    }));
}

// (of either type: 16-bit units have more places, 32-bit ones are more)
size_t bias_backward_workspace_bytes(const BiasRequest &r) {
    return std::max(partial_bytes(backward_args(r, 4)), partial_bytes(backward_args(r, 8))) +
           align_up(static_cast<size_t>(r.H) * (2 * r.far + 1) * 4, 256);
}

int bias_backward_run(const BiasRequest &r) {
    const size_t need = bias_backward_workspace_bytes(r);
    if (need > 0 && (!r.workspace || r.workspace_bytes < need || reinterpret_cast<uintptr_t>(r.workspace) % 256 != 0))
        return PLE_E_WORKSPACE;
    BiasArgs a = backward_args(r, r.out_dtype == PLE_DTYPE_F32 ? 4 : 8);
    a.total = reinterpret_cast<float *>(static_cast<char *>(r.workspace) + partial_bytes(a));
    const dim3 grid(static_cast<unsigned>(std::min((a.tiles + kWavesPerBlock - 1) / kWavesPerBlock, kMaxGrid)));
    const int64_t blocks = r.H * ((2 * r.far + 1 + kWave - 1) / kWave);
    const hipError_t rc = with_type(r.out_dtype, [&](auto t) {
        constexpr int T = decltype(t)::value;
        if (a.tiles > 0) {
            if (a.k < vec_elems<T>())
                hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_bias_backward_kernel<T, true>), grid, dim3(kBlock), 0, r.stream, a);
            else
                hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_bias_backward_kernel<T, false>), grid, dim3(kBlock), 0, r.stream, a);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_bias_total_kernel<T>), dim3(static_cast<unsigned>(std::min(blocks, kMaxGrid))),
                           dim3(kJoinThreads), 0, r.stream, a);
        return hipGetLastError();
    });
    if (rc != hipSuccess) return static_cast<int>(rc);
    const int64_t units = r.H * ((r.R + kJoinRows - 1) / kJoinRows);
    hipLaunchKernelGGL(ple_bias_join_kernel, dim3(static_cast<unsigned>(std::min(units, kMaxGrid))), dim3(kJoinThreads), 0, r.stream, a);
    return static_cast<int>(hipGetLastError());
}

}  // namespace ple

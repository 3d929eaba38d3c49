// Embedding lookup with scaling, and its gradient by sorted tokens (gfx950).
//
// Forward: out[i, :] = round(scale * W[row(i), :]), where row(i) is the token,
// or offsets[f] + token for column f of categorical tokens [N, F].  A negative
// token is a missing value (a row of zeros), a token beyond its table gives a
// row of NaN; neither reads the table.
//
// Backward: dW[r, :] = round(scale * sum_{i: row(i) = r} g[i, :]), rows without
// tokens 0.  The tokens are sorted by row with a stable radix sort (the order
// of equal rows is the tokens' own), the sorted list is cut into chunks of S
// tokens, and each chunk adds up its runs of equal rows in registers: a run
// inside one chunk is a finished row, one that crosses a chunk's border leaves
// a partial sum in 32 bits, and a last kernel adds a run's partials in order.
// So however unevenly the tokens are spread, every chunk is the same work, and
// the order of every sum is fixed: no atomics on floating-point data.

#include <algorithm>

#include "ple_internal.h"
#include "ple_rows.h"

namespace ple {
namespace {

constexpr int kSortBlock = 512;
constexpr int kSortWaves = kSortBlock / kWave;
constexpr int kMaxDigitBits = 10;
constexpr int kMaxTiles = 256;
constexpr int kMinTile = 1024;         // tokens a sorting workgroup takes at least

struct TokenArgs {
    const void *tokens;
    const int64_t *offsets;      // NULL: one table
    int64_t V, padding;
    uint32_t T, F;
    int wide;                    // 64-bit tokens
};

constexpr int64_t kMissing = -1;
constexpr int64_t kBeyond = -2;

// Row of token i, kMissing or kBeyond.
__device__ __forceinline__ int64_t token_row(const TokenArgs &a, uint32_t i) {
    const int64_t tok = a.wide ? static_cast<const int64_t *>(a.tokens)[i] : static_cast<const int32_t *>(a.tokens)[i];
    int64_t lo = 0, n = a.V;
    if (a.offsets) {
        const uint32_t f = i % a.F;
        lo = a.offsets[f];
        n = a.offsets[f + 1] - lo;
    }
    if (tok < 0) return kMissing;
    return tok < n && lo >= 0 && lo < a.V && tok < a.V - lo ? lo + tok : kBeyond;
}

// Sort key of token i: its row, or V for a token that has no gradient.
__device__ __forceinline__ uint32_t token_key(const TokenArgs &a, uint32_t i) {
    const int64_t tok = a.wide ? static_cast<const int64_t *>(a.tokens)[i] : static_cast<const int32_t *>(a.tokens)[i];
    const int64_t row = token_row(a, i);
    return static_cast<uint32_t>(row < 0 || (a.padding >= 0 && tok == a.padding) ? a.V : row);
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------

struct GatherArgs {
    TokenArgs t;
    const void *weight;
    void *out;
    int64_t D;
    float scale;
    int lg;                      // log2 of the lanes that share a token
};

constexpr int kGatherUnroll = 4;

template <int W, int O, int VEC>
__global__ __launch_bounds__(kBlock) void ple_lookup_kernel(GatherArgs a) {
    const int lanes = 1 << a.lg;
    const int64_t i = (static_cast<int64_t>(blockIdx.x) << (8 - a.lg)) + (threadIdx.x >> a.lg);
    if (i >= a.t.T) return;
    const int64_t row = token_row(a.t, static_cast<uint32_t>(i));
    const int64_t col0 = (static_cast<int64_t>(blockIdx.y) * kGatherUnroll * lanes + (threadIdx.x & (lanes - 1))) * VEC;
    float v[kGatherUnroll][VEC];
#pragma unroll
    for (int u = 0; u < kGatherUnroll; ++u) {
        const int64_t col = col0 + static_cast<int64_t>(u) * lanes * VEC;
        if (row >= 0 && col < a.D) {
            load_vec<W, VEC>(a.weight, row * a.D + col, v[u]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[u][e] *= a.scale;
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[u][e] = row == kBeyond ? __builtin_nanf("") : 0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < kGatherUnroll; ++u) {
        const int64_t col = col0 + static_cast<int64_t>(u) * lanes * VEC;
        if (col < a.D) store_vec<O, VEC>(a.out, i * a.D + col, v[u]);
    }
}

// ---------------------------------------------------------------------------
// backward: the sort
// ---------------------------------------------------------------------------

struct SortArgs {
    TokenArgs t;
    const uint32_t *keys_in, *pos_in;    // the first pass makes them from the tokens
    uint32_t *keys_out, *pos_out;
    uint32_t *counts;                    // [tiles, 1 << bits]
    uint8_t *present;                    // [V]: rows that have tokens
    uint32_t tile;                       // tokens a workgroup takes
    int tiles, shift, bits;
};

template <bool FIRST>
__device__ __forceinline__ uint32_t sort_key(const SortArgs &a, uint32_t i) {
    if constexpr (FIRST) return token_key(a.t, i);
    else return a.keys_in[i];
}

template <bool FIRST>
__global__ __launch_bounds__(kSortBlock) void ple_lookup_count_kernel(SortArgs a) {
    __shared__ uint32_t hist[1 << kMaxDigitBits];
    const uint32_t digits = 1u << a.bits;
    for (uint32_t d = threadIdx.x; d < digits; d += kSortBlock) hist[d] = 0;
    if constexpr (FIRST)
        for (int64_t r = static_cast<int64_t>(blockIdx.x) * kSortBlock + threadIdx.x; r < a.t.V;
             r += static_cast<int64_t>(gridDim.x) * kSortBlock)
            a.present[r] = 0;
    __syncthreads();
    const uint64_t begin = static_cast<uint64_t>(blockIdx.x) * a.tile;
    const uint64_t end = begin + a.tile < a.t.T ? begin + a.tile : a.t.T;
    for (uint64_t i = begin + threadIdx.x; i < end; i += kSortBlock)
        atomicAdd(&hist[(sort_key<FIRST>(a, static_cast<uint32_t>(i)) >> a.shift) & (digits - 1)], 1u);
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < digits; d += kSortBlock)
        a.counts[static_cast<size_t>(blockIdx.x) * digits + d] = hist[d];
}

// Each wave takes a contiguous part of the workgroup's tile, 64 tokens at a
// time: the lanes with the same digit find each other by ballots, and their
// places are the wave's running offset of that digit plus their rank.
template <bool FIRST, bool LAST>
__global__ __launch_bounds__(kSortBlock) void ple_lookup_scatter_kernel(SortArgs a) {
    extern __shared__ uint32_t s_off[];      // [kSortWaves][digits]
    __shared__ uint32_t s_wave[kSortWaves];
    const uint32_t digits = 1u << a.bits;
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
    for (uint32_t d = tid; d < kSortWaves * digits; d += kSortBlock) s_off[d] = 0;
    __syncthreads();
    const uint64_t begin = static_cast<uint64_t>(blockIdx.x) * a.tile;
    const uint64_t end = begin + a.tile < a.t.T ? begin + a.tile : a.t.T;
    const uint32_t part = a.tile / kSortWaves;      // (a multiple of 64)
    const uint64_t w0 = begin + static_cast<uint64_t>(wave) * part;
    const uint64_t w1 = w0 + part < end ? w0 + part : end;
    uint32_t *mine = s_off + wave * digits;
    for (uint64_t i = w0 + lane; i < w1; i += kWave)
        atomicAdd(&mine[(sort_key<FIRST>(a, static_cast<uint32_t>(i)) >> a.shift) & (digits - 1)], 1u);

    // the digits of this thread: `per` adjacent ones
    const uint32_t per = digits > kSortBlock ? digits / kSortBlock : 1;
    uint32_t before[4] = {0, 0, 0, 0}, total[4] = {0, 0, 0, 0}, sum = 0;
    if (tid * per < digits) {
        for (int t = 0; t < a.tiles; ++t)
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (k < per) {
                    const uint32_t c = a.counts[static_cast<size_t>(t) * digits + tid * per + k];
                    total[k] += c;
                    if (t < static_cast<int>(blockIdx.x)) before[k] += c;
                }
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) sum += total[k];
    }
    // tokens of smaller digits: exclusive sum over the threads
    uint32_t incl = sum;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const uint32_t up = __shfl_up(incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == kWave - 1) s_wave[wave] = incl;
    __syncthreads();
    uint32_t base = incl - sum;
    for (int w = 0; w < wave; ++w) base += s_wave[w];
    if (tid * per < digits) {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            if (k < per) {
                uint32_t at = base + before[k];
                for (int w = 0; w < kSortWaves; ++w) {
                    uint32_t *p = &s_off[w * digits + tid * per + k];
                    const uint32_t c = *p;
                    *p = at;
                    at += c;
                }
                base += total[k];
            }
    }
    __syncthreads();

    volatile uint32_t *off = mine;
    for (uint64_t i0 = w0; i0 < w1; i0 += kWave) {
        const uint64_t i = i0 + lane;
        const bool on = i < w1;
        const uint32_t key = on ? sort_key<FIRST>(a, static_cast<uint32_t>(i)) : 0;
        const uint32_t digit = (key >> a.shift) & (digits - 1);
        uint64_t same = __ballot(on);
        for (int b = 0; b < a.bits; ++b) {
            const bool bit = (digit >> b) & 1;
            const uint64_t set = __ballot(bit);
            same &= bit ? set : ~set;
        }
        const uint32_t rank = __popcll(same & ((uint64_t{1} << lane) - 1));
        uint32_t dst = 0;
        if (on) dst = off[digit] + rank;
        __builtin_amdgcn_wave_barrier();
        if (on && rank == 0) off[digit] = dst + __popcll(same);
        __builtin_amdgcn_wave_barrier();
        if (on) {
            a.keys_out[dst] = key;
            a.pos_out[dst] = FIRST ? static_cast<uint32_t>(i) : a.pos_in[i];
            if (LAST && key < static_cast<uint64_t>(a.t.V)) a.present[key] = 1;
        }
    }
}

// ---------------------------------------------------------------------------
// backward: sums over runs of equal rows
// ---------------------------------------------------------------------------

struct SumArgs {
    const void *g;
    const uint32_t *keys, *pos;
    const uint8_t *present;              // NULL: no row has tokens
    float *partial;                      // [chunks, 2, D]
    void *dw;
    int64_t D, V;
    uint32_t T, S, chunks;
    int lg, colblocks;
    uint32_t sum_blocks, zero_rows;      // workgroups that sum; rows a zeroing one looks at
    float scale;
};

constexpr int kSumUnroll = 8;

template <int O, int VEC>
__device__ __forceinline__ void store_row(const SumArgs &a, uint32_t row, int64_t col, const float *acc) {
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = acc[e] * a.scale;
    store_vec<O, VEC>(a.dw, static_cast<int64_t>(row) * a.D + col, v);
}

template <int G, int O, int VEC>
__global__ __launch_bounds__(kBlock) void ple_lookup_sum_kernel(SumArgs a) {
    if (blockIdx.x >= a.sum_blocks) {
        // rows without tokens
        const int64_t r0 = static_cast<int64_t>(blockIdx.x - a.sum_blocks) * a.zero_rows;
        const uint32_t rows = static_cast<uint32_t>(a.V - r0 < a.zero_rows ? a.V - r0 : a.zero_rows);
        const uint32_t vecs = static_cast<uint32_t>(a.D / VEC);
        const float zero[VEC] = {};
        for (uint32_t j = threadIdx.x; j < rows * vecs; j += kBlock) {
            const uint32_t r = j / vecs;
            if (!a.present || !a.present[r0 + r])
                store_vec<O, VEC>(a.dw, (r0 + r) * a.D + static_cast<int64_t>(j - r * vecs) * VEC, zero);
        }
        return;
    }
    const int lanes = 1 << a.lg;
    const uint32_t unit = (blockIdx.x << (8 - a.lg)) + (threadIdx.x >> a.lg);
    const uint32_t chunk = unit / a.colblocks;
    const int64_t col = (static_cast<int64_t>(unit % a.colblocks) * lanes + (threadIdx.x & (lanes - 1))) * VEC;
    if (chunk >= a.chunks || col >= a.D) return;
    const uint32_t begin = chunk * a.S;
    const uint32_t end = a.T - begin < a.S ? a.T : begin + a.S;
    uint32_t cur = a.keys[begin];
    bool first = true, joined = begin > 0 && a.keys[begin - 1] == cur;
    float acc[VEC] = {};
    const auto flush = [&](bool ended) {
        if (cur >= static_cast<uint64_t>(a.V)) return;
        if (!joined && ended) store_row<O, VEC>(a, cur, col, acc);
        else store_vec<PLE_DTYPE_F32, VEC>(a.partial, (static_cast<int64_t>(chunk) * 2 + (first ? 0 : 1)) * a.D + col, acc);
    };
    for (uint32_t i = begin; i < end; i += kSumUnroll) {
        uint32_t key[kSumUnroll];
        float v[kSumUnroll][VEC];
#pragma unroll
        for (int u = 0; u < kSumUnroll; ++u) {
            const uint32_t at = i + u < end ? i + u : end - 1;
            key[u] = a.keys[at];
            load_vec<G, VEC>(a.g, static_cast<int64_t>(a.pos[at]) * a.D + col, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kSumUnroll; ++u) {
            if (i + u >= end) break;
            if (key[u] != cur) {
                flush(true);
                cur = key[u];
                first = joined = false;
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += v[u][e];
        }
    }
    flush(!(end < a.T && a.keys[end] == cur));
}

// Runs that cross a chunk's border: the workgroup of the chunk where the run
// starts adds its partials, the groups of lanes a contiguous part each.
template <int O, int VEC>
__global__ __launch_bounds__(kBlock) void ple_lookup_join_kernel(SumArgs a) {
    __shared__ float s_sum[kBlock * VEC];
    const uint32_t chunk = blockIdx.x / a.colblocks;
    const uint32_t begin = chunk * a.S;
    if (a.T - begin <= a.S) return;      // (the last chunk: nothing follows)
    const uint32_t end = begin + a.S;
    const uint32_t key = a.keys[end];
    if (key >= static_cast<uint64_t>(a.V) || a.keys[end - 1] != key) return;
    const bool whole = a.keys[begin] == key;
    if (whole && begin > 0 && a.keys[begin - 1] == key) return;     // it started before
    // chunks that begin inside the run: chunk + 1 .. last
    uint32_t stop = chunk + 1;
    for (;;) {
        const uint32_t c = stop + threadIdx.x % kWave;
        const uint64_t out = __ballot(!(c < a.chunks && a.keys[c * a.S] == key));
        if (out) {
            stop += __builtin_ctzll(out);
            break;
        }
        stop += kWave;
    }
    const int lanes = 1 << a.lg, teams = kBlock >> a.lg;
    const int team = threadIdx.x >> a.lg, lane = threadIdx.x & (lanes - 1);
    const int64_t col = (static_cast<int64_t>(blockIdx.x % a.colblocks) * lanes + lane) * VEC;
    const uint32_t n = stop - chunk, per = (n + teams - 1) / teams;
    float acc[VEC] = {};
    if (col < a.D) {
        const uint32_t p1 = (team + 1) * per < n ? (team + 1) * per : n;
#pragma unroll 4
        for (uint32_t p = team * per; p < p1; ++p) {
            float v[VEC];
            const int64_t slot = static_cast<int64_t>(chunk + p) * 2 + (p == 0 && !whole ? 1 : 0);
            load_vec<PLE_DTYPE_F32, VEC>(a.partial, slot * a.D + col, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += v[e];
        }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) s_sum[e * kBlock + threadIdx.x] = acc[e];
    __syncthreads();
    if (team == 0 && col < a.D) {
        for (int t = 1; t < teams; ++t)
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += s_sum[e * kBlock + t * lanes + lane];
        store_row<O, VEC>(a, key, col, acc);
    }
}

// ---------------------------------------------------------------------------
// plans and launches
// ---------------------------------------------------------------------------

int bits_of(uint64_t v) { return v == 0 ? 0 : 64 - __builtin_clzll(v); }

// Widest vector (8, 4, 2 or 1 elements) that rows of D elements allow and every
// address is aligned for (16 bytes at most).
int row_vec(int64_t D, std::initializer_list<std::pair<const void *, int>> ptrs) {
    for (int vec = 8; vec > 1; vec /= 2) {
        bool ok = D % vec == 0;
        for (const auto &[p, dtype] : ptrs)
            ok = ok && reinterpret_cast<uintptr_t>(p) % std::min(16, vec * elem_bytes(dtype)) == 0;
        if (ok) return vec;
    }
    return 1;
}

struct SumPlan {
    int passes, bits, tiles, lg, colblocks;
    uint32_t tile, S, chunks;
    size_t o_pos, o_keys2, o_pos2, o_counts, o_present, o_partial, bytes;
};

SumPlan plan_sum(int64_t T, int64_t V, int64_t D, int vec) {
    SumPlan p{};
    const int key_bits = std::max(1, bits_of(static_cast<uint64_t>(V)));
    p.passes = (key_bits + kMaxDigitBits - 1) / kMaxDigitBits;
    p.bits = (key_bits + p.passes - 1) / p.passes;
    const int64_t per = (T + kMaxTiles - 1) / kMaxTiles;
    p.tile = static_cast<uint32_t>(std::max<int64_t>(kMinTile, (per + kSortBlock - 1) / kSortBlock * kSortBlock));
    p.tiles = static_cast<int>((T + p.tile - 1) / p.tile);
    const int64_t vecs = (D + vec - 1) / vec;
    p.lg = std::min(6, vecs <= 1 ? 0 : bits_of(static_cast<uint64_t>(vecs - 1)));
    p.colblocks = static_cast<int>((vecs + (int64_t{1} << p.lg) - 1) >> p.lg);
    p.S = 32;
    p.chunks = static_cast<uint32_t>((T + p.S - 1) / p.S);
    const size_t list = align_up(static_cast<size_t>(T) * 4, 256);
    size_t at = list;
    const auto take = [&](size_t n) {
        const size_t o = at;
        at += align_up(n, 256);
        return o;
    };
    p.o_pos = take(list);
    p.o_keys2 = take(p.passes > 1 ? list : 0);
    p.o_pos2 = take(p.passes > 1 ? list : 0);
    p.o_counts = take(static_cast<size_t>(p.tiles) * 4 << p.bits);
    p.o_present = take(static_cast<size_t>(V));
    p.o_partial = take(static_cast<size_t>(p.chunks) * 2 * D * 4);
    p.bytes = at;
    return p;
}

template <int W, int O, int VEC>
hipError_t launch_gather(GatherArgs a, hipStream_t s) {
    const int64_t vecs = a.D / VEC;
    a.lg = std::min(6, vecs <= 1 ? 0 : bits_of(static_cast<uint64_t>(vecs - 1)));
    const int64_t per_block = kBlock >> a.lg, cols = (int64_t{1} << a.lg) * kGatherUnroll;
    const dim3 grid(static_cast<unsigned>((a.t.T + per_block - 1) / per_block),
                    static_cast<unsigned>((vecs + cols - 1) / cols));
    hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_kernel<W, O, VEC>), grid, dim3(kBlock), 0, s, a);
    return hipGetLastError();
}

template <int G, int O, int VEC>
hipError_t launch_sum(SumArgs a, hipStream_t s) {
    const uint64_t units = static_cast<uint64_t>(a.chunks) * a.colblocks, per_block = kBlock >> a.lg;
    a.sum_blocks = static_cast<uint32_t>((units + per_block - 1) / per_block);
    const int64_t row_bytes = a.D * elem_bytes(O);
    a.zero_rows = static_cast<uint32_t>(std::max<int64_t>(1, 32768 / row_bytes));
    const uint64_t zero_blocks = (a.V + a.zero_rows - 1) / a.zero_rows;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_sum_kernel<G, O, VEC>),
                       dim3(static_cast<unsigned>(a.sum_blocks + zero_blocks)), dim3(kBlock), 0, s, a);
    if (a.chunks > 1)
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_join_kernel<O, VEC>), dim3(a.chunks * a.colblocks), dim3(kBlock),
                           0, s, a);
    return hipGetLastError();
}

// f(integral_constant<int, dtype>) for a dtype known at run time
template <typename F>
hipError_t with_dtype(int dtype, F f) {
    switch (dtype) {
        case PLE_DTYPE_F32: return f(std::integral_constant<int, PLE_DTYPE_F32>{});
        case PLE_DTYPE_F16: return f(std::integral_constant<int, PLE_DTYPE_F16>{});
        default: return f(std::integral_constant<int, PLE_DTYPE_BF16>{});
    }
}

template <typename F>
hipError_t with_vec(int vec, F f) {
    switch (vec) {
        case 8: return f(std::integral_constant<int, 8>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 2: return f(std::integral_constant<int, 2>{});
        default: return f(std::integral_constant<int, 1>{});
    }
}

TokenArgs token_args(const LookupRequest &r) {
    TokenArgs t{};
    t.tokens = r.tokens;
    t.offsets = r.offsets;
    t.V = r.V;
    t.padding = r.padding;
    t.T = static_cast<uint32_t>(r.T);
    t.F = static_cast<uint32_t>(r.F);
    t.wide = r.wide;
    return t;
}

}  // namespace

int lookup_run(const LookupRequest &r) {
    GatherArgs a{};
    a.t = token_args(r);
    a.weight = r.table;
    a.out = r.out;
    a.D = r.D;
    a.scale = r.scale;
    const int vec = row_vec(r.D, {{r.table, r.table_dtype}, {r.out, r.out_dtype}});
    return static_cast<int>(with_dtype(r.table_dtype, [&](auto w) {
        return with_dtype(r.out_dtype, [&](auto o) {
            return with_vec(vec, [&](auto v) {
                return launch_gather<decltype(w)::value, decltype(o)::value, decltype(v)::value>(a, r.stream);
            });
        });
    }));
}

size_t lookup_backward_workspace_bytes(int64_t T, int64_t V, int64_t D) { return T == 0 ? 0 : plan_sum(T, V, D, 1).bytes; }

int lookup_backward_run(const LookupRequest &r) {
    const int vec = row_vec(r.D, {{r.grad, r.out_dtype}, {r.dw, r.table_dtype}});
    const SumPlan p = plan_sum(std::max<int64_t>(r.T, 0), r.V, r.D, vec);
    if (r.T > 0 && (!r.workspace || r.workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(r.workspace) % 256 != 0))
        return PLE_E_WORKSPACE;
    char *ws = static_cast<char *>(r.workspace);
    const auto list = [&](size_t o) { return reinterpret_cast<uint32_t *>(ws + o); };
    SortArgs s{};
    s.t = token_args(r);
    s.tile = p.tile;
    s.tiles = p.tiles;
    s.bits = p.bits;
    SumArgs a{};
    if (r.T > 0) {
        s.counts = list(p.o_counts);
        s.present = reinterpret_cast<uint8_t *>(ws + p.o_present);
        uint32_t *keys[2] = {list(0), p.passes > 1 ? list(p.o_keys2) : nullptr};
        uint32_t *pos[2] = {list(p.o_pos), p.passes > 1 ? list(p.o_pos2) : nullptr};
        const size_t lds = static_cast<size_t>(kSortWaves) * 4 << p.bits;
        const dim3 grid(p.tiles), block(kSortBlock);
        for (int k = 0; k < p.passes; ++k) {
            s.shift = k * p.bits;
            s.keys_in = keys[(k + 1) & 1];
            s.pos_in = pos[(k + 1) & 1];
            s.keys_out = keys[k & 1];
            s.pos_out = pos[k & 1];
            const bool last = k + 1 == p.passes;
            if (k == 0) {
                hipLaunchKernelGGL(ple_lookup_count_kernel<true>, grid, block, 0, r.stream, s);
                if (last) hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_scatter_kernel<true, true>), grid, block, lds, r.stream, s);
                else hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_scatter_kernel<true, false>), grid, block, lds, r.stream, s);
            } else {
                hipLaunchKernelGGL(ple_lookup_count_kernel<false>, grid, block, 0, r.stream, s);
                if (last) hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_scatter_kernel<false, true>), grid, block, lds, r.stream, s);
                else hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_scatter_kernel<false, false>), grid, block, lds, r.stream, s);
            }
        }
        a.keys = s.keys_out;
        a.pos = s.pos_out;
        a.present = s.present;
        a.partial = reinterpret_cast<float *>(ws + p.o_partial);
    }
    a.g = r.grad;
    a.dw = r.dw;
    a.D = r.D;
    a.V = r.V;
    a.T = static_cast<uint32_t>(r.T);
    a.S = p.S;
    a.chunks = p.chunks;
    a.lg = p.lg;
    a.colblocks = p.colblocks;
    a.scale = r.scale;
    return static_cast<int>(with_dtype(r.out_dtype, [&](auto g) {
        return with_dtype(r.table_dtype, [&](auto o) {
            return with_vec(vec, [&](auto v) {
                return launch_sum<decltype(g)::value, decltype(o)::value, decltype(v)::value>(a, r.stream);
            });
        });
    }));
}

}  // namespace ple

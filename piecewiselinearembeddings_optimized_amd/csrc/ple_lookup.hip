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
//
// Measured (one MI355X): 65536 tokens x 2048 bf16 over 131072 rows, 1.17 GB in
// all, 251 us: forward 78 us (its reads and stores, 4.7 TB/s), sort 30 us of
// which 14 beside the rows that are cleared, clearing and sums 150 us (805 MB,
// 5.4 TB/s), joins 5 us.  196608 categories x 32 fp32: 52 us, of which the sort's
// four launches 31 (each a chain of loads, ranks and barriers, on few workgroups)
// and the sums 14.

#include <algorithm>

#include "ple_internal.h"
#include "ple_rows.h"

namespace ple {
namespace {

constexpr int kMaxDigitBits = 10;
constexpr int kMaxTiles = 256;

// A sorting workgroup by its digits' bits (8 or 10 at most).  Up to 8 bits 16 waves
// rank a token a lane at a time, the shortest chain (by 8 waves of 4 tokens 55.0
// against 52.5 us, 196608 x 32, and 53.6 against 50.6, 16384 x 1024: whole
// backwards with their forwards); beyond, every wave's counts are 4 KB, and 8 waves
// leave room for the workgroups that clear rows beside them (65536 x 2048: 251.8
// against 254.5 us).
template <int BITS>
struct Sort {
    static constexpr int kBlock = BITS <= 8 ? 1024 : 512;
    static constexpr int kWaves = kBlock / kWave;
    static constexpr int kRounds = BITS <= 8 ? 1 : 4;    // tokens a lane ranks at a time
    static constexpr int kStep = kBlock * kRounds;
};
// One workgroup sorts up to this many tokens by itself, in LDS: its 16 waves
// hold up to 8 of them a lane (one launch for four; whole backwards of rows of 64:
// 1500 tokens 14.5 us, by several workgroups 22.8; 4096 19.3 and 23.6; 8000 25.3 and
// 24.4 to 25.6, and 27.9 against 32.9 where it clears 100000 rows of 256 meanwhile;
// 16384 tokens' sort alone takes one workgroup 38).
constexpr int kLocalBlock = 1024;
constexpr int kLocalWaves = kLocalBlock / kWave;
constexpr int kLocalRounds = 8;
constexpr int64_t kLocalTokens = kLocalBlock * kLocalRounds;

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
    int64_t D, first;            // first: the launch's first token
    float scale;
    int lg;                      // log2 of the lanes that share a token
};

constexpr int kGatherUnroll = 4;
constexpr int64_t kGatherBlocks = 1 << 23;       // of a launch: a grid holds fewer than 2^32 threads a dimension

// A group of lanes has kGatherUnroll vectors in flight: of one token's row
// where it is long enough, else of as many tokens' rows (TOKENS).  The output is
// stored past the caches: the next pass's reads find the memory-side cache free
// of its lines (16384 x 1024 12.5 -> 10 us, 65536 x 2048 91 -> 79 us; 196608 x 32
// as fast either way).
template <int W, int O, int VEC, bool TOKENS>
__global__ __launch_bounds__(kBlock) void ple_lookup_kernel(GatherArgs a) {
    const int lanes = 1 << a.lg;
    const int64_t per_block = kBlock >> a.lg;
    const int64_t i0 = a.first + static_cast<int64_t>(blockIdx.x) * per_block * (TOKENS ? kGatherUnroll : 1) +
                       (threadIdx.x >> a.lg);
    const int64_t col0 = (static_cast<int64_t>(blockIdx.y) * (TOKENS ? 1 : kGatherUnroll) * lanes +
                          (threadIdx.x & (lanes - 1))) * VEC;
    const auto token = [&](int u) { return i0 + (TOKENS ? u * per_block : 0); };
    const auto column = [&](int u) { return col0 + (TOKENS ? 0 : static_cast<int64_t>(u) * lanes * VEC); };
    int64_t row[kGatherUnroll];
#pragma unroll
    for (int u = 0; u < kGatherUnroll; ++u)
        row[u] = TOKENS || u == 0 ? (token(u) < a.t.T ? token_row(a.t, static_cast<uint32_t>(token(u))) : kMissing) : row[0];
    float v[kGatherUnroll][VEC];
#pragma unroll
    for (int u = 0; u < kGatherUnroll; ++u) {
        if (row[u] >= 0 && column(u) < a.D) {
            load_vec<W, VEC>(a.weight, row[u] * a.D + column(u), v[u]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[u][e] = row[u] == kBeyond ? __builtin_nanf("") : 0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < kGatherUnroll; ++u) {
        if (token(u) >= a.t.T || column(u) >= a.D) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[u][e] *= a.scale;
        store_vec<O, VEC, true>(a.out, token(u) * a.D + column(u), v[u]);
    }
}

// ---------------------------------------------------------------------------
// backward: the sort
// ---------------------------------------------------------------------------

// Rows without tokens are written by workgroups of their own beside the sort's,
// which leave the memory idle: `present` tells them which rows those are, or
// (NULL) every row is cleared and the rows with tokens are written again.
struct ZeroArgs {
    char *dw;
    const uint8_t *present;
    int64_t begin, end;          // rows
    uint32_t units, rows;        // units of a row; rows a workgroup looks at
    int unit;                    // bytes: 16, 4 or 2
};

// (Stored past the caches: beside a gradient of more than the memory-side cache,
// plain stores of the rows and of the zeros took 288 us where these take 251,
// 65536 tokens x 2048 over 131072 rows; smaller ones are as fast either way.)
__device__ __forceinline__ void zero_rows(const ZeroArgs &z, int64_t block) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const int64_t r0 = z.begin + block * z.rows;
    const uint32_t rows = static_cast<uint32_t>(z.end - r0 < z.rows ? z.end - r0 : z.rows);
    for (uint32_t j = threadIdx.x; j < rows * z.units; j += blockDim.x) {
        if (z.present && z.present[r0 + j / z.units]) continue;
        char *p = z.dw + (r0 * z.units + j) * z.unit;
        if (z.unit == 16) __builtin_nontemporal_store(u32x4{0, 0, 0, 0}, reinterpret_cast<u32x4 *>(p));
        else if (z.unit == 4) *reinterpret_cast<uint32_t *>(p) = 0;
        else *reinterpret_cast<uint16_t *>(p) = 0;
    }
}

struct SortArgs {
    TokenArgs t;
    ZeroArgs z;                          // of the launch's workgroups past `tiles`
    uint32_t *keys_in;                   // the first pass's count kernel makes them from the tokens
    const uint32_t *pos_in;              // first pass: the tokens' own order
    uint32_t *keys_out, *pos_out;
    uint32_t *counts;                    // [tiles, 1 << bits]
    uint8_t *present;                    // [V]: rows that have tokens
    uint32_t tile;                       // tokens a workgroup takes
    int tiles, shift, bits, passes;
};

// The lanes of the wave that are `on` and have this lane's digit, of at most
// BITS bits: a ballot for each bit, whose mask or its complement every lane
// keeps by its own bit.  (Bits above the digit are 0 for all and keep all.)
template <int BITS>
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, bool on) {
    const uint64_t all = __ballot(on);
    uint32_t lo = static_cast<uint32_t>(all), hi = static_cast<uint32_t>(all >> 32);
#pragma unroll
    for (int b = 0; b < BITS; ++b) {
        const uint32_t mine = static_cast<uint32_t>(static_cast<int32_t>(digit << (31 - b)) >> 31);   // all ones: bit set
        const uint64_t set = __ballot(mine != 0);
        lo &= ~(static_cast<uint32_t>(set) ^ mine);
        hi &= ~(static_cast<uint32_t>(set >> 32) ^ mine);
    }
    return (static_cast<uint64_t>(hi) << 32) | lo;
}

// Rank of this lane's token among the wave's tokens of its digit so far, whose
// number `seen` holds (in LDS, the wave's own).
template <int BITS, typename Count>
__device__ __forceinline__ uint32_t rank_token(volatile Count *seen, uint32_t digit, bool on) {
    const uint32_t prior = seen[digit];
    const uint64_t same = same_digit<BITS>(digit, on);
    const uint32_t below = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(same >> 32),
                                                     __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(same), 0));
    __builtin_amdgcn_wave_barrier();
    if (on && below == 0) seen[digit] = static_cast<Count>(prior + __popcll(same));
    __builtin_amdgcn_wave_barrier();
    return prior + below;
}

// Exclusive sums over the workgroup's threads of one value each.
template <int THREADS>
__device__ __forceinline__ uint32_t exclusive_sum(uint32_t v, uint32_t *s_wave) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    uint32_t incl = v;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const uint32_t up = __shfl_up(incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == kWave - 1) s_wave[wave] = incl;
    __syncthreads();
    uint32_t base = incl - v;
    for (int w = 0; w < wave; ++w) base += s_wave[w];
    return base;
}

template <bool FIRST, int BITS>
__global__ __launch_bounds__(Sort<BITS>::kBlock) void ple_lookup_count_kernel(SortArgs a) {
    constexpr int kSortBlock = Sort<BITS>::kBlock, kSortRounds = Sort<BITS>::kRounds, kSortStep = Sort<BITS>::kStep;
    __shared__ uint32_t hist[1 << BITS];
    if (static_cast<int>(blockIdx.x) >= a.tiles) {
        zero_rows(a.z, blockIdx.x - a.tiles);
        return;
    }
    const uint32_t digits = 1u << a.bits;
    for (uint32_t d = threadIdx.x; d < digits; d += kSortBlock) hist[d] = 0;
    if constexpr (FIRST)
        // (`present` is rounded up to 16 bytes)
        for (int64_t r = static_cast<int64_t>(blockIdx.x) * kSortBlock + threadIdx.x; r < (a.t.V + 15) / 16;
             r += static_cast<int64_t>(a.tiles) * kSortBlock)
            reinterpret_cast<uint4 *>(a.present)[r] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const uint64_t begin = static_cast<uint64_t>(blockIdx.x) * a.tile;
    const uint64_t end = begin + a.tile < a.t.T ? begin + a.tile : a.t.T;
    for (uint64_t i0 = begin + threadIdx.x; i0 < end; i0 += kSortStep) {
        uint32_t key[kSortRounds];
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r) {
            const uint64_t i = i0 + r * kSortBlock;
            if constexpr (FIRST) key[r] = token_key(a.t, static_cast<uint32_t>(i < end ? i : end - 1));
            else key[r] = a.keys_in[i < end ? i : end - 1];
        }
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r)
            if (i0 + r * kSortBlock < end) {
                if constexpr (FIRST) a.keys_in[i0 + r * kSortBlock] = key[r];
                atomicAdd(&hist[(key[r] >> a.shift) & (digits - 1)], 1u);
            }
    }
    __syncthreads();
    for (uint32_t d = threadIdx.x; d < digits; d += kSortBlock)
        a.counts[static_cast<size_t>(blockIdx.x) * digits + d] = hist[d];
}

// The workgroup's first place of every digit comes from all workgroups' counts
// (each reads them all, 16 bytes a load and the loads in parallel: a kernel of
// its own for these sums costs more than the reads up to 256 workgroups).  Then
// it walks its tokens in steps: each wave takes a contiguous part of a step and
// ranks its tokens per digit, the waves' numbers give each wave its place.
template <bool FIRST, int BITS>
__global__ __launch_bounds__(Sort<BITS>::kBlock) void ple_lookup_scatter_kernel(SortArgs a) {
    constexpr int kSortBlock = Sort<BITS>::kBlock, kSortWaves = Sort<BITS>::kWaves, kSortRounds = Sort<BITS>::kRounds;
    constexpr int kSortStep = Sort<BITS>::kStep;
    extern __shared__ uint32_t s_dyn[];
    __shared__ uint32_t s_wave[kSortWaves];
    if (static_cast<int>(blockIdx.x) >= a.tiles) {
        zero_rows(a.z, blockIdx.x - a.tiles);
        return;
    }
    const uint32_t digits = 1u << a.bits;
    uint32_t *s_place = s_dyn, *s_total = s_dyn + digits, *s_seen = s_dyn + 2 * digits;   // seen: [waves, digits]
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
    const uint64_t begin = static_cast<uint64_t>(blockIdx.x) * a.tile;
    const uint64_t end = begin + a.tile < a.t.T ? begin + a.tile : a.t.T;
    uint32_t key[kSortRounds], pos[kSortRounds], rank[kSortRounds];
    uint64_t i0 = begin + wave * (kWave * kSortRounds) + lane;
    const auto load = [&] {
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r) {
            const uint64_t i = i0 + r * kWave < end ? i0 + r * kWave : end - 1;
            key[r] = a.keys_in[i];
            pos[r] = FIRST ? static_cast<uint32_t>(i) : a.pos_in[i];
        }
    };
    load();
    for (uint32_t d = tid; d < (2 + kSortWaves) * digits; d += kSortBlock) s_dyn[d] = 0;
    __syncthreads();
    {
        const uint32_t wide = digits / 4;            // (at least 1: bits >= 2)
        const uint32_t groups = kSortBlock / wide;
        const uint32_t group = tid / wide, at = tid % wide;
        uint32_t before[4] = {0, 0, 0, 0}, total[4] = {0, 0, 0, 0};
#pragma unroll 8
        for (uint32_t t = group; t < static_cast<uint32_t>(a.tiles); t += groups) {
            const uint4 c = reinterpret_cast<const uint4 *>(a.counts)[static_cast<size_t>(t) * wide + at];
            const uint32_t mine = t < blockIdx.x ? ~0u : 0u;
            total[0] += c.x; total[1] += c.y; total[2] += c.z; total[3] += c.w;
            before[0] += c.x & mine; before[1] += c.y & mine; before[2] += c.z & mine; before[3] += c.w & mine;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            atomicAdd(&s_place[4 * at + k], before[k]);
            atomicAdd(&s_total[4 * at + k], total[k]);
        }
    }
    uint32_t *mine = s_seen + wave * digits;
    const auto rank_step = [&] {
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r)
            rank[r] = rank_token<BITS, uint32_t>(mine, (key[r] >> a.shift) & (digits - 1), i0 + r * kWave < end);
    };
    rank_step();
    __syncthreads();
    {
        constexpr int kPer = ((1 << BITS) + kSortBlock - 1) / kSortBlock;
        uint32_t total[kPer], sum = 0;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const uint32_t d = tid * kPer + k;
            total[k] = d < digits ? s_total[d] : 0;
            sum += total[k];
        }
        uint32_t base = exclusive_sum<kSortBlock>(sum, s_wave);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const uint32_t d = tid * kPer + k;
            if (d < digits) s_place[d] += base;
            base += total[k];
        }
    }
    for (uint64_t step = begin;;) {
        __syncthreads();
        for (uint32_t d = tid; d < digits; d += kSortBlock) {
            uint32_t at = s_place[d];
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) {
                const uint32_t c = s_seen[w * digits + d];
                s_seen[w * digits + d] = at;
                at += c;
            }
            s_place[d] = at;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kSortRounds; ++r)
            if (i0 + r * kWave < end) {
                const uint32_t dst = mine[(key[r] >> a.shift) & (digits - 1)] + rank[r];
                a.keys_out[dst] = key[r];
                a.pos_out[dst] = pos[r];
                if (FIRST && key[r] < static_cast<uint64_t>(a.t.V)) a.present[key[r]] = 1;
            }
        step += kSortStep;
        if (step >= end) break;
        i0 += kSortStep;
        load();
        __syncthreads();       // (the places of the step before are used)
        for (uint32_t d = tid; d < kSortWaves * digits; d += kSortBlock) s_seen[d] = 0;
        __syncthreads();
        rank_step();
    }
}

// All passes for up to kLocalTokens tokens in one workgroup: keys and positions
// go through LDS between the passes, ranks as above.
template <int ROUNDS, int BITS>
__global__ __launch_bounds__(kLocalBlock) void ple_lookup_sort_kernel(SortArgs a) {
    extern __shared__ uint32_t s_dyn[];
    __shared__ uint32_t s_wave[kLocalWaves];
    if (blockIdx.x > 0) {
        zero_rows(a.z, blockIdx.x - 1);
        return;
    }
    const uint32_t digits = 1u << a.bits, T = a.t.T;
    uint32_t *s_key = s_dyn;                                             // [rounded T]
    const uint32_t room = (T + kLocalBlock - 1) / kLocalBlock * kLocalBlock;
    uint16_t *s_pos = reinterpret_cast<uint16_t *>(s_key + room);        // [rounded T]
    uint16_t *s_seen = s_pos + room;                                     // [waves, digits]
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
    const int rounds = static_cast<int>(room / kLocalBlock);             // (at most ROUNDS)
    const uint32_t i0 = wave * rounds * kWave + lane;
    uint32_t key[ROUNDS], pos[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
        if (r < rounds) {
            const uint32_t i = i0 + r * kWave < T ? i0 + r * kWave : T - 1;
            key[r] = token_key(a.t, i);
            pos[r] = i;
        }
    // (`present` is rounded up to 16 bytes; NULL: this launch clears all rows)
    for (int64_t r = tid; a.present && r < (a.t.V + 15) / 16; r += kLocalBlock)
        reinterpret_cast<uint4 *>(a.present)[r] = make_uint4(0, 0, 0, 0);
    uint16_t *mine = s_seen + wave * digits;
    for (int pass = 0; pass < a.passes; ++pass) {
        const int shift = pass * a.bits;
        for (uint32_t d = tid; d < kLocalWaves * digits / 2; d += kLocalBlock) reinterpret_cast<uint32_t *>(s_seen)[d] = 0;
        __syncthreads();
        uint32_t rank[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (r < rounds)
                rank[r] = rank_token<BITS, uint16_t>(mine, (key[r] >> shift) & (digits - 1), i0 + r * kWave < T);
        __syncthreads();
        // (digits <= kLocalBlock: one a thread)
        uint32_t seen[kLocalWaves], sum = 0;
        if (tid < static_cast<int>(digits))
#pragma unroll
            for (int w = 0; w < kLocalWaves; ++w) {
                seen[w] = s_seen[w * digits + tid];
                sum += seen[w];
            }
        uint32_t at = exclusive_sum<kLocalBlock>(sum, s_wave);
        if (tid < static_cast<int>(digits))
#pragma unroll
            for (int w = 0; w < kLocalWaves; ++w) {
                s_seen[w * digits + tid] = static_cast<uint16_t>(at);
                at += seen[w];
            }
        __syncthreads();
        const bool last = pass + 1 == a.passes;
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (r < rounds && i0 + r * kWave < T) {
                const uint32_t dst = mine[(key[r] >> shift) & (digits - 1)] + rank[r];
                s_key[dst] = key[r];
                s_pos[dst] = static_cast<uint16_t>(pos[r]);
            }
        __syncthreads();
        if (!last) {
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r)
                if (r < rounds && i0 + r * kWave < T) {
                    key[r] = s_key[i0 + r * kWave];
                    pos[r] = s_pos[i0 + r * kWave];
                }
        }
    }
    for (uint32_t i = tid; i < T; i += kLocalBlock) {
        const uint32_t k = s_key[i];
        a.keys_out[i] = k;
        a.pos_out[i] = s_pos[i];
        if (a.present && k < static_cast<uint64_t>(a.t.V)) a.present[k] = 1;
    }
}

// ---------------------------------------------------------------------------
// backward: sums over runs of equal rows
// ---------------------------------------------------------------------------

struct SumArgs {
    const void *g;
    const uint32_t *keys, *pos;
    ZeroArgs z;                          // of the launch's workgroups past `sum_blocks`
    float *partial;                      // [blocks, 2, D]: a run from the block before, a run into the next
    void *dw;
    int64_t D, V;
    uint32_t T, S, block, blocks;        // tokens a group of lanes, a workgroup takes; workgroups (a block of columns)
    int lg, colblocks;
    uint32_t sum_blocks;                 // workgroups that sum
    float scale;
};

constexpr int kSumUnroll = 8;

template <int O, int VEC>
__device__ __forceinline__ void store_row(const SumArgs &a, uint32_t row, int64_t col, const float *acc) {
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = acc[e] * a.scale;
    store_vec<O, VEC, true>(a.dw, static_cast<int64_t>(row) * a.D + col, v);
}

template <int VEC>
__device__ __forceinline__ void store_partial(const SumArgs &a, uint32_t block, int slot, int64_t col, const float *acc) {
    store_vec<PLE_DTYPE_F32, VEC>(a.partial, (static_cast<int64_t>(block) * 2 + slot) * a.D + col, acc);
}

// A group of lanes adds up its S tokens' runs in registers.  A run inside them is
// finished; the sums of one that came from the group before (the head) and of
// one that goes on in the next (the tail) meet in LDS, and those that cross the
// workgroup's border become partials.
template <int G, int O, int VEC>
__global__ __launch_bounds__(kBlock) void ple_lookup_sum_kernel(SumArgs a) {
    if (blockIdx.x >= a.sum_blocks) {
        zero_rows(a.z, blockIdx.x - a.sum_blocks);
        return;
    }
    enum { kHead = 1, kThrough = 2, kTail = 4 };     // through: the head goes on into the next group
    __shared__ float s_head[kBlock * VEC];
    __shared__ int s_has[kBlock];
    const int lanes = 1 << a.lg, teams = kBlock >> a.lg;
    const int team = threadIdx.x >> a.lg, lane = threadIdx.x & (lanes - 1);
    const uint32_t block = blockIdx.x / a.colblocks;
    const int64_t col = (static_cast<int64_t>(blockIdx.x % a.colblocks) * lanes + lane) * VEC;
    const uint64_t begin = static_cast<uint64_t>(block) * a.block + static_cast<uint64_t>(team) * a.S;
    const uint64_t end = begin + a.S < a.T ? begin + a.S : a.T;
    float acc[VEC] = {};
    uint32_t cur = 0;
    int has = 0;
    if (begin < a.T && col < a.D) {
        cur = a.keys[begin];
        bool joined = begin > 0 && a.keys[begin - 1] == cur;
        const auto end_run = [&] {
            if (cur < static_cast<uint64_t>(a.V)) {
                if (joined) {
                    has |= kHead;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) s_head[e * kBlock + threadIdx.x] = acc[e];
                } else {
                    store_row<O, VEC>(a, cur, col, acc);
                }
            }
        };
        for (uint64_t i = begin; i < end; i += kSumUnroll) {
            uint32_t key[kSumUnroll];
            float v[kSumUnroll][VEC];
#pragma unroll
            for (int u = 0; u < kSumUnroll; ++u) {
                const uint64_t at = i + u < end ? i + u : end - 1;
                key[u] = a.keys[at];
                load_vec<G, VEC>(a.g, static_cast<int64_t>(a.pos[at]) * a.D + col, v[u]);
            }
#pragma unroll
            for (int u = 0; u < kSumUnroll; ++u) {
                if (i + u >= end) break;
                if (key[u] != cur) {
                    end_run();
                    cur = key[u];
                    joined = false;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += v[u][e];
            }
        }
        if (end < a.T && a.keys[end] == cur) {
            if (cur < static_cast<uint64_t>(a.V)) {
                if (joined) {
                    end_run();
                    has |= kThrough;
                } else {
                    has |= kTail;
                }
            }
        } else {
            end_run();
        }
    }
    // head[t] += head[t + 1] for as long as the run goes through, by doubling: then
    // a head has the whole rest of its run, and kThrough says that it leaves the
    // workgroup
    if (lane == 0) s_has[team] = has;        // (lane 0's columns exist)
    const int through = __syncthreads_or(has & kThrough);
    for (int d = 1; through && d < teams; d *= 2) {
        const bool on = (s_has[team] & kThrough) && team + d < teams;
        const int other = on ? s_has[team + d] : 0;
        float v[VEC];
        if (on)
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = s_head[e * kBlock + threadIdx.x] + s_head[e * kBlock + threadIdx.x + d * lanes];
        __syncthreads();
        if (on) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) s_head[e * kBlock + threadIdx.x] = v[e];
            if (lane == 0 && !(other & kThrough)) s_has[team] &= ~kThrough;
        }
        __syncthreads();
    }
    if (col >= a.D) return;
    if (has & kTail) {
        bool leaves = true;
        if (team + 1 < teams) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += s_head[e * kBlock + threadIdx.x + lanes];
            leaves = s_has[team + 1] & kThrough;
        }
        if (leaves) store_partial<VEC>(a, block, 1, col, acc);
        else store_row<O, VEC>(a, cur, col, acc);
    }
    if (team == 0 && (has & kHead)) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = s_head[e * kBlock + lane];
        store_partial<VEC>(a, block, 0, col, acc);
    }
}

// Runs that cross a block's border.  A group of lanes looks at one block: a run
// that starts there and goes on in up to kShortRun blocks it adds itself.  A
// longer one the workgroup adds, its groups a contiguous part each; it looks at
// no more than kShortRun blocks, so it has one of those at most.
constexpr int kShortRun = 8;

template <int O, int VEC>
__global__ __launch_bounds__(kBlock) void ple_lookup_join_kernel(SumArgs a) {
    __shared__ float s_sum[kBlock * VEC];
    __shared__ uint32_t s_long;              // the long run's block
    const int lanes = 1 << a.lg, teams = kBlock >> a.lg;
    const int team = threadIdx.x >> a.lg, lane = threadIdx.x & (lanes - 1);
    const int looking = teams < kShortRun ? teams : kShortRun;
    const uint32_t block = blockIdx.x / a.colblocks * looking + team;
    const int64_t col = (static_cast<int64_t>(blockIdx.x % a.colblocks) * lanes + lane) * VEC;
    const auto first_key = [&](uint32_t b) { return a.keys[static_cast<uint64_t>(b) * a.block]; };
    uint32_t n = 0, key = 0;                 // n: partials of the run that starts here
    if (team < looking && block + 1 < a.blocks) {    // (the last block has nothing behind it)
        const uint64_t begin = static_cast<uint64_t>(block) * a.block;
        uint32_t ahead[kShortRun + 1];
#pragma unroll
        for (uint32_t j = 0; j <= kShortRun; ++j)
            ahead[j] = first_key(block + 1 + j < a.blocks ? block + 1 + j : a.blocks - 1);
        const uint32_t last = a.keys[begin + a.block - 1], first = a.keys[begin];
        const uint32_t prior = begin > 0 ? a.keys[begin - 1] : ~0u;      // (no key is ~0)
        key = ahead[0];
        if (key < static_cast<uint64_t>(a.V) && last == key && !(first == key && prior == key)) {
            n = 2;
#pragma unroll
            for (uint32_t j = 1; j <= kShortRun; ++j)
                if (n == j + 1 && block + 1 + j < a.blocks && ahead[j] == key) n = j + 2;
        }
    }
    const bool more = n > kShortRun + 1;
    if (n > 0 && !more && col < a.D) {
        float acc[VEC];
        load_vec<PLE_DTYPE_F32, VEC>(a.partial, (static_cast<int64_t>(block) * 2 + 1) * a.D + col, acc);
#pragma unroll
        for (uint32_t p = 1; p <= kShortRun; ++p)
            if (p < n) {
                float v[VEC];
                load_vec<PLE_DTYPE_F32, VEC>(a.partial, static_cast<int64_t>(block + p) * 2 * a.D + col, v);
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += v[e];
            }
        store_row<O, VEC>(a, key, col, acc);
    }
    if (more && lane == 0) s_long = block;
    if (!__syncthreads_or(more)) return;
    const uint32_t at = s_long, k = first_key(at + 1);
    // blocks that begin inside the run: at + 1 .. stop - 1
    uint32_t stop = at + kShortRun + 1;
    for (;;) {
        const uint32_t b = stop + threadIdx.x % kWave;
        const uint64_t out = __ballot(!(b < a.blocks && first_key(b) == k));
        if (out) {
            stop += __builtin_ctzll(out);
            break;
        }
        stop += kWave;
    }
    const uint32_t parts = stop - at, per = (parts + teams - 1) / teams;
    float acc[VEC] = {};
    if (col < a.D) {
        const uint32_t p1 = (team + 1) * per < parts ? (team + 1) * per : parts;
#pragma unroll 8
        for (uint32_t p = team * per; p < p1; ++p) {
            float v[VEC];
            load_vec<PLE_DTYPE_F32, VEC>(a.partial, (static_cast<int64_t>(at + p) * 2 + (p == 0 ? 1 : 0)) * a.D + col, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += v[e];
        }
    }
    for (int half = teams / 2; half > 0; half /= 2) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) s_sum[e * kBlock + threadIdx.x] = acc[e];
        __syncthreads();
        if (team < half)
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += s_sum[e * kBlock + threadIdx.x + half * lanes];
        __syncthreads();
    }
    if (team == 0 && col < a.D) store_row<O, VEC>(a, k, col, acc);
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
    uint32_t tile, S, block, blocks;     // block: tokens a summing workgroup takes
    size_t o_pos, o_keys2, o_pos2, o_counts, o_present, o_partial, bytes;
};

SumPlan plan_sum(int64_t T, int64_t V, int64_t D, int vec) {
    SumPlan p{};
    const int key_bits = std::max(1, bits_of(static_cast<uint64_t>(V)));
    p.passes = (key_bits + kMaxDigitBits - 1) / kMaxDigitBits;
    p.bits = (key_bits + p.passes - 1) / p.passes;
    p.bits = std::max(2, p.bits);        // (counts are read four digits at a time)
    const int64_t per = (T + kMaxTiles - 1) / kMaxTiles, step = p.bits <= 8 ? Sort<8>::kStep : Sort<kMaxDigitBits>::kStep;
    p.tile = static_cast<uint32_t>(std::max<int64_t>(1, (per + step - 1) / step) * step);
    p.tiles = static_cast<int>((T + p.tile - 1) / p.tile);
    const int64_t vecs = (D + vec - 1) / vec;
    p.lg = std::min(6, vecs <= 1 ? 0 : bits_of(static_cast<uint64_t>(vecs - 1)));
    p.colblocks = static_cast<int>((vecs + (int64_t{1} << p.lg) - 1) >> p.lg);
    // tokens a chunk: enough waves for the GPU (16 a CU, 8 elements a lane), chunks
    // long enough for their partials to be few.  (By T and D alone, which size the
    // workspace.)
    const int64_t waves = T * D / (8 * kWave);
    p.S = 8;
    while (p.S < 128 && waves / p.S > 16 * 256) p.S *= 2;
    p.block = p.S * (kBlock >> p.lg);
    p.blocks = static_cast<uint32_t>((T + p.block - 1) / p.block);
    // (partials: by the fewest tokens a block has, those of rows of 64 lanes)
    const size_t most_blocks = static_cast<size_t>((T + p.S * kWavesPerBlock - 1) / (p.S * kWavesPerBlock));
    const size_t list = align_up(static_cast<size_t>(T) * 4, 256);
    size_t at = list;
    const auto take = [&](size_t n) {
        const size_t o = at;
        at += align_up(n, 256);
        return o;
    };
    p.o_pos = take(list);
    p.o_keys2 = take(list);
    p.o_pos2 = take(p.passes > 1 ? list : 0);
    p.o_counts = take(static_cast<size_t>(p.tiles) * 4 << p.bits);
    p.o_present = take(static_cast<size_t>(V));
    p.o_partial = take(most_blocks * 2 * D * 4);
    p.bytes = at;
    return p;
}

uint32_t zero_blocks(const ZeroArgs &z) {
    return z.end > z.begin ? static_cast<uint32_t>((z.end - z.begin + z.rows - 1) / z.rows) : 0;
}

template <int W, int O, int VEC>
hipError_t launch_gather(GatherArgs a, hipStream_t s) {
    const int64_t vecs = a.D / VEC;
    a.lg = std::min(6, vecs <= 1 ? 0 : bits_of(static_cast<uint64_t>(vecs - 1)));
    const int64_t per_block = kBlock >> a.lg, lanes = int64_t{1} << a.lg;
    const auto blocks = [](int64_t n, int64_t per) { return static_cast<unsigned>((n + per - 1) / per); };
    const int64_t per = vecs <= lanes ? per_block * kGatherUnroll : per_block;
    for (a.first = 0; a.first < a.t.T; a.first += kGatherBlocks * per) {
        const unsigned n = static_cast<unsigned>(std::min(kGatherBlocks, (a.t.T - a.first + per - 1) / per));
        if (vecs <= lanes)
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_kernel<W, O, VEC, true>), dim3(n), dim3(kBlock), 0, s, a);
        else
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_kernel<W, O, VEC, false>), dim3(n, blocks(vecs, lanes * kGatherUnroll)),
                               dim3(kBlock), 0, s, a);
    }
    return hipGetLastError();
}

template <int G, int O, int VEC>
hipError_t launch_sum(SumArgs a, hipStream_t s) {
    a.sum_blocks = a.blocks * a.colblocks;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_sum_kernel<G, O, VEC>), dim3(a.sum_blocks + zero_blocks(a.z)), dim3(kBlock), 0,
                       s, a);
    if (a.blocks > 1) {
        const uint32_t looking = std::min(kBlock >> a.lg, kShortRun);
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_join_kernel<O, VEC>), dim3((a.blocks + looking - 1) / looking * a.colblocks),
                           dim3(kBlock), 0, s, a);
    }
    return hipGetLastError();
}

constexpr int64_t kClearBlocks = 1 << 21;        // of a launch, beside its others: a grid holds fewer than 2^32 threads

struct ClearPlan {
    uint32_t rows;                       // a workgroup looks at
    bool local;                          // one workgroup sorts
    bool all;                            // rows with tokens too
    bool in_sort;                        // by the sort's launches, else by the sum's
};

ClearPlan plan_clear(const SumPlan &p, int64_t T, int64_t V, int64_t row_bytes) {
    ClearPlan c{};
    // 32 KB a workgroup, or as many rows as keep a launch's workgroups few enough
    c.rows = static_cast<uint32_t>(std::max<int64_t>({1, 32768 / row_bytes, (V + kClearBlocks - 1) / kClearBlocks}));
    c.local = T > 0 && T <= kLocalTokens;
    // the sort of one workgroup takes as long as clearing some 100 MB; clearing
    // rows that have tokens too is little where they are few
    c.all = c.local && V >= 4 * T;
    c.in_sort = c.local ? c.all : T > 0 && p.passes > 1;
    return c;
}

// Threads of the largest grid of a backward's launches.
int64_t most_threads(const SumPlan &p, const ClearPlan &c, int64_t T, int64_t V) {
    const int64_t clear = (V + c.rows - 1) / c.rows;
    const int64_t sort = T == 0 ? 0 : (c.local ? 1 : p.tiles) + (c.in_sort ? clear : 0);
    const int64_t sum = static_cast<int64_t>(p.blocks) * p.colblocks + (c.in_sort ? 0 : clear);
    const int block = c.local ? kLocalBlock : p.bits <= 8 ? Sort<8>::kBlock : Sort<kMaxDigitBits>::kBlock;
    return std::max(sort * block, sum * kBlock);
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

template <int BITS>
hipError_t launch_local_sort(const SortArgs &s, hipStream_t stream) {
    const size_t room = align_up(s.t.T, kLocalBlock);
    const size_t lds = room * 6 + (static_cast<size_t>(kLocalWaves) * 2 << s.bits);
    const dim3 grid(1 + zero_blocks(s.z)), block(kLocalBlock);
    if (room <= 2 * kLocalBlock)
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_sort_kernel<2, BITS>), grid, block, lds, stream, s);
    else
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_sort_kernel<kLocalRounds, BITS>), grid, block, lds, stream, s);
    return hipGetLastError();
}

// One pass; the second one's two kernels clear a third and two thirds of `rows`
// rows (their own times are about as 1 to 2).
template <int BITS>
hipError_t launch_sort_pass(SortArgs s, int pass, int64_t rows, hipStream_t stream) {
    const size_t lds = static_cast<size_t>(2 + Sort<BITS>::kWaves) * 4 << s.bits;
    const dim3 block(Sort<BITS>::kBlock);
    s.z.begin = 0;
    s.z.end = pass == 1 ? rows / 3 : 0;
    const auto grid = [&] { return dim3(s.tiles + zero_blocks(s.z)); };
    if (pass == 0) hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_count_kernel<true, BITS>), grid(), block, 0, stream, s);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_count_kernel<false, BITS>), grid(), block, 0, stream, s);
    const hipError_t rc = hipGetLastError();
    if (rc != hipSuccess) return rc;
    s.z.begin = s.z.end;
    s.z.end = pass == 1 ? rows : 0;
    if (pass == 0) hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_scatter_kernel<true, BITS>), grid(), block, lds, stream, s);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_lookup_scatter_kernel<false, BITS>), grid(), block, lds, stream, s);
    return hipGetLastError();
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

int lookup_backward_plan_info(const LookupRequest &r, ple_lookup_plan_info_t *info) {
    const int vec = row_vec(r.D, {{r.grad, r.out_dtype}, {r.dw, r.table_dtype}});
    const SumPlan p = plan_sum(r.T, r.V, r.D, vec);
    const ClearPlan c = plan_clear(p, r.T, r.V, r.D * elem_bytes(r.table_dtype));
    const int64_t most = most_threads(p, c, r.T, r.V);
    if (most >= int64_t{1} << 32) return PLE_E_TOO_LARGE;
    *info = ple_lookup_plan_info_t{};
    info->one_workgroup = c.local;
    info->passes = r.T > 0 ? p.passes : 0;
    info->digit_bits = r.T > 0 ? p.bits : 0;
    info->sort_workgroups = r.T == 0 ? 0 : c.local ? 1 : p.tiles;
    info->sum_workgroups = static_cast<int64_t>(p.blocks) * p.colblocks;
    info->clear_rows = c.rows;
    info->most_threads = most;
    info->workspace_bytes = r.T > 0 ? p.bytes : 0;
    return PLE_OK;
}

int lookup_backward_run(const LookupRequest &r) {
    const int vec = row_vec(r.D, {{r.grad, r.out_dtype}, {r.dw, r.table_dtype}});
    const SumPlan p = plan_sum(r.T, r.V, r.D, vec);
    if (r.T > 0 && (!r.workspace || r.workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(r.workspace) % 256 != 0))
        return PLE_E_WORKSPACE;
    const int64_t row_bytes = r.D * elem_bytes(r.table_dtype);
    const ClearPlan clear = plan_clear(p, r.T, r.V, row_bytes);
    // (beyond the memory of any device: the sums' threads are fewer than a gradient's elements)
    if (most_threads(p, clear, r.T, r.V) >= int64_t{1} << 32) return PLE_E_TOO_LARGE;
    char *ws = static_cast<char *>(r.workspace);
    const auto list = [&](size_t o) { return reinterpret_cast<uint32_t *>(ws + o); };
    SortArgs s{};
    s.t = token_args(r);
    s.tile = p.tile;
    s.tiles = p.tiles;
    s.bits = p.bits;
    SumArgs a{};
    ZeroArgs z{};
    z.dw = static_cast<char *>(r.dw);
    z.unit = reinterpret_cast<uintptr_t>(r.dw) % 16 == 0 && row_bytes % 16 == 0 ? 16 : elem_bytes(r.table_dtype);
    z.units = static_cast<uint32_t>(row_bytes / z.unit);
    z.rows = clear.rows;
    z.end = r.V;
    a.z = z;
    if (clear.in_sort) a.z.end = 0;
    if (r.T > 0) {
        s.counts = list(p.o_counts);
        s.present = reinterpret_cast<uint8_t *>(ws + p.o_present);
        a.z.present = s.present;
        uint32_t *keys[2] = {list(0), list(p.o_keys2)};
        uint32_t *pos[2] = {list(p.o_pos), p.passes > 1 ? list(p.o_pos2) : nullptr};
        s.passes = p.passes;
        s.z = z;
        // (the sums read what the sort wrote: nothing follows a sort that was not launched)
        hipError_t rc = hipSuccess;
        if (clear.local) {
            s.keys_out = keys[0];
            s.pos_out = pos[0];
            if (clear.all) s.present = nullptr;
            else s.z.end = 0;
            rc = p.bits <= 8 ? launch_local_sort<8>(s, r.stream) : launch_local_sort<kMaxDigitBits>(s, r.stream);
        } else {
            s.z.present = s.present;
            for (int k = 0; k < p.passes && rc == hipSuccess; ++k) {
                s.shift = k * p.bits;
                s.keys_in = keys[(k + 1) & 1];
                s.pos_in = pos[(k + 1) & 1];
                s.keys_out = keys[k & 1];
                s.pos_out = pos[k & 1];
                rc = p.bits <= 8 ? launch_sort_pass<8>(s, k, r.V, r.stream) : launch_sort_pass<kMaxDigitBits>(s, k, r.V, r.stream);
            }
        }
        if (rc != hipSuccess) return static_cast<int>(rc);
        a.keys = s.keys_out;
        a.pos = s.pos_out;
        a.partial = reinterpret_cast<float *>(ws + p.o_partial);
    }
    a.g = r.grad;
    a.dw = r.dw;
    a.D = r.D;
    a.V = r.V;
    a.T = static_cast<uint32_t>(r.T);
    a.S = p.S;
    a.block = p.block;
    a.blocks = p.blocks;
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

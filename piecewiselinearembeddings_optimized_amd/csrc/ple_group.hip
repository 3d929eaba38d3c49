// Group norm with an activation, channels last (gfx950).  For a sample of S rows
// (features, pixels) of C channels in G groups of P = C / G adjacent ones, every
// group of a sample over its S P values:
//
//     m = mean x,  rho = 1 / sqrt(mean (x - m)^2 + eps)
//     z = (x - m) rho w_c + b_c,  y = act(z)
//
// Backward, with xh = (x - m) rho, dz = dy act'(z), g = dz w_c:
//
//     dw_c = sum dz xh, db_c = sum dz            over samples and rows
//     dx = rho (g - mean g - xh mean(g xh))      means over the group
//
// Bound by memory: forward a read and a write, backward two reads and a write.
// A lane's vector of 16 bytes is the same channels in every row it takes, so
// parameters, per-channel sums and (groups of whole vectors) the group are the
// lane's own.
//
// Held form: a workgroup holds a sample's groups (all, or a slab of them) in
// registers: statistics in two passes over the registers, one read of memory.
// Shared form, for samples that several workgroups hold: each publishes what it knows
// of a group and takes the others'.  A value is its own flag (a 64-bit word that is
// not kUnknown), so nothing has to be ordered; and a workgroup that does not find
// another's in time reads that one's rows and computes it, so no wait depends on what
// else runs.
// Split form, for samples larger still: sums of pieces of rows (per channel, the
// squares about the piece's own mean), a join per group, and a second read that
// applies it.
//
// Measured, forward / backward: held, 16384 x 64 x 64 fp32 100 / 155 us (5.4 / 5.2 TB/s);
// shared, 8 x 65536 x 256 bf16 140 / 241 us (3.8 / 3.3 TB/s: three workgroups a CU load,
// wait for each other and store in step) and 16 x 4096 x 320 27 / 49 us; split, 1 x
// 200000 x 960 288 / 440 us (2.7 / 2.6 TB/s: x, and the gradient, are read twice).

#include <algorithm>

#include "ple_internal.h"
#include "ple_rows.h"

namespace ple {
namespace {

// A lane's piece of a row: W dwords, or (W 0) one 16-bit element.
template <int T, int W>
struct Piece {
    static constexpr int kElems = W == 0 ? 1 : (T == PLE_DTYPE_F32 ? W : 2 * W);
    static constexpr int kWords = W == 0 ? 1 : W;
    uint32_t w[kWords];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load(const void *p, int64_t i) { load_at(static_cast<const char *>(p) + i * elem_bytes(T)); }
    __device__ __forceinline__ void load_at(const char *q) {
        if constexpr (W == 4) {
            const uint4 v = *reinterpret_cast<const uint4 *>(q);
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else if constexpr (W == 1) {
            w[0] = *reinterpret_cast<const uint32_t *>(q);
        } else {
            w[0] = *reinterpret_cast<const uint16_t *>(q);
        }
    }
    __device__ __forceinline__ float operator[](int e) const { return grad_elem<T>(w, e); }
    // Keeps the piece as it was loaded: without it the compiler widens 16-bit elements
    // where they are loaded and keeps them all, twice the registers.
    __device__ __forceinline__ void keep() {
        if constexpr (T != PLE_DTYPE_F32)
#pragma unroll
            for (int i = 0; i < kWords; ++i) asm volatile("" : "+v"(w[i]));
    }
};

template <int T, int W>
__device__ __forceinline__ void store_piece(void *p, int64_t i, const float *v) {
    store_out<T, Piece<T, W>::kElems, false>(p, i, v);
}

// A sample's rows (or its groups' values in them) in shares of one size, the last one
// smaller.  The host makes the inverses: kernels here divide no floats.  (With divisions in
// the fold's loop its squares were wrong, other ones each time, wherever two of its waves
// shared a SIMD.  Seen in its code: several divisions interleaved, a v_div_fmas with its VCC
// from an s_mov right before it.  That this was the cause is not shown; with the inverses
// the squares are right.)
struct Shares {
    float count, count_last, inv, inv_last;
    int last;                    // the last share
    __device__ __forceinline__ float inverse(int share) const { return share == last ? inv_last : inv; }
    // the squared distance of a share's mean (its sum's), for each of its values
    __device__ __forceinline__ float distance(float sum, int share, float mean) const {
        const float d = sum * inverse(share) - mean;
        return (share == last ? count_last : count) * d * d;
    }
};

struct GroupArgs {
    const void *x, *g, *weight, *bias;
    void *y;                     // forward: y; backward: dx
    float2 *stats;               // [N, G]: mean and factor
    float2 *sums;                // split: [N, pieces, C] sums of a piece's channels
    float2 *channels;            // split backward: [N, C]
    float2 *means;               // split backward: [N, G]
    float *partial;              // backward: [parts, 2, C] sums of dz and of dz xh
    int64_t N, S, blocks;        // blocks: units of work of a slab
    int C, G, P;
    int L, slots, A, U;          // lanes of a row, rows at once of a sample, lanes of a sample, samples at once
    int slabs, Cs, Gs;           // slabs of a row, channels and groups of one
    int team;                    // lanes that join a group
    uint32_t wide_inverse;       // 2^32 / values of a group in a row, rounded up
    int pieces;                  // split: pieces of a sample
    int folded;                  // split: pieces after the fold
    Shares share, fold;          // shared: values of a member; split: rows of a piece, of folded ones
    float2 *folds;               // split: [N, folded, C]
    uint64_t *exchange;          // shared: [units, members, Gs] what the members know of a group
    int members, member_rows;    // shared: workgroups of a unit, rows of each
    int polls;                   // shared: how often a member looks for another's
    int act, param_dtype, param_vectors;
    float eps, inv;              // inv: 1 / (S P)
};

// ---------------------------------------------------------------------------
// activations
// ---------------------------------------------------------------------------

// (What workgroups compute in each other's place, and what the backward repeats of the
// forward, has to have the same bits wherever it is compiled: such products and sums are
// fused by fmaf, or not at all.)

// Standard normal distribution and density at z.  Abramowitz and Stegun 26.2.17: the
// tail is the density times a polynomial in 1 / (1 + p |z|), off by at most 7.5e-8.
__device__ __forceinline__ void normal_cdf(float z, float &cdf, float &pdf) {
#pragma clang fp contract(off)
    pdf = 0.39894228f * __expf(-0.5f * z * z);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.2316419f, fabsf(z), 1.0f));
    const float tail = pdf * t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.330274429f, -1.821255978f), 1.781477937f), -0.356563782f), 0.319381530f);
    cdf = z > 0.0f ? 1.0f - tail : tail;
}

__device__ __forceinline__ float logistic(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

template <int E>
__device__ __forceinline__ void activate(float (&z)[E], int act) {
    if (act == PLE_ACT_RELU) {
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] = z[e] < 0.0f ? 0.0f : z[e];         // (NaN stays)
    } else if (act == PLE_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] *= logistic(z[e]);
    } else if (act == PLE_ACT_GELU) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float cdf, pdf;
            normal_cdf(z[e], cdf, pdf);
            z[e] *= cdf;
        }
    }
}

// act'(z) in place of z
template <int E>
__device__ __forceinline__ void slopes(float (&z)[E], int act) {
    if (act == PLE_ACT_RELU) {
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] = z[e] > 0.0f ? 1.0f : (z[e] <= 0.0f ? 0.0f : z[e]);
    } else if (act == PLE_ACT_SILU) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float s = logistic(z[e]);
            z[e] = fmaf(z[e] * s, 1.0f - s, s);
        }
    } else if (act == PLE_ACT_GELU) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float cdf, pdf;
            normal_cdf(z[e], cdf, pdf);
            z[e] = fmaf(z[e], pdf, cdf);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] = 1.0f;
    }
}

// ---------------------------------------------------------------------------
// held form
// ---------------------------------------------------------------------------

// A lane's place in its workgroup: sample, row slot and piece of the row.
struct Place {
    int unit, slot, lane, thread;
    bool on;
    // The same, as values that the compiler takes for new ones in every turn of a loop:
    // it would else compute the addresses of a turn before the loop, and hold them all.
    __device__ __forceinline__ Place again() const {
        Place q = *this;
        asm volatile("" : "+v"(q.unit), "+v"(q.slot), "+v"(q.lane), "+v"(q.thread));
        return q;
    }
    __device__ __forceinline__ explicit Place(const GroupArgs &a) : thread(threadIdx.x) {
        unit = threadIdx.x / a.A;
        const int r = threadIdx.x - unit * a.A;
        slot = r / a.L;
        lane = r - slot * a.L;
        on = unit < a.U;
    }
};

// A lane's E values of a parameter from channel c0 on (`none` without one).
template <int E>
__device__ __forceinline__ void load_params(const GroupArgs &a, const void *p, int c0, float none, float (&v)[E]) {
    if (!p) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = none;
    } else if (E >= 4 && a.param_vectors) {
        if (a.param_dtype == PLE_DTYPE_F32) load_vec<PLE_DTYPE_F32, E>(p, c0, v);
        else if (a.param_dtype == PLE_DTYPE_BF16) load_vec<PLE_DTYPE_BF16, E>(p, c0, v);
        else load_vec<PLE_DTYPE_F16, E>(p, c0, v);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = c0 + e < a.C ? load_any(p, c0 + e, a.param_dtype) : none;
    }
}

// The slab's parameters as 32-bit values in LDS, weights then biases.
template <int THREADS>
__device__ __forceinline__ void stage_params(const GroupArgs &a, int slab, float *s_params) {
    for (int c = threadIdx.x; c < a.Cs; c += THREADS) {
        s_params[c] = a.weight ? load_any(a.weight, slab * a.Cs + c, a.param_dtype) : 1.0f;
        s_params[a.Cs + c] = a.bias ? load_any(a.bias, slab * a.Cs + c, a.param_dtype) : 0.0f;
    }
}

template <int E>
__device__ __forceinline__ void staged(const float *p, float (&v)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = p[e];
}

// A value that the compiler takes for another in every turn of a loop: it would else
// make a copy of the loop for each activation, and hold what all of them need.
__device__ __forceinline__ int unhoisted(int v) {
    asm volatile("" : "+s"(v));
    return v;
}

// The groups of a lane's channels (WHOLE: one group for the whole piece).
template <int E, bool WHOLE>
struct Groups {
    static constexpr int kEach = WHOLE ? 1 : E;
    int first;
    uint32_t starts;             // bit e: channel e is the first of a group (e > 0)
    __device__ __forceinline__ Groups again() const {
        Groups q = *this;
        asm volatile("" : "+v"(q.first), "+v"(q.starts));
        return q;
    }
    __device__ __forceinline__ Groups(const GroupArgs &a, int channel) {
        first = channel / a.P;
        starts = 0;
        if constexpr (!WHOLE) {
            int r = channel - first * a.P;
#pragma unroll
            for (int e = 1; e < E; ++e)
                if (++r == a.P) {
                    r = 0;
                    starts |= 1u << e;
                }
        }
    }
    __device__ __forceinline__ int of(int e) const { return WHOLE ? first : first + __popc(starts & ((2u << e) - 1)); }
};

// A lane's values that are joined lie in LDS by value, its workgroup's lanes next to each
// other (a few places more than lanes, so that a group's channels are in other banks).
template <int THREADS>
constexpr int kPlane = THREADS + 8;

// Joins the workgroup's values in LDS (WHOLE: one a lane, else one a channel) over each
// group: a team of lanes adds a group's, and `done(group, sums)` runs on the team's
// first lane.  K values are joined at once.
template <int K, int E, bool WHOLE, int THREADS, typename F>
__device__ __forceinline__ void join_lds(const GroupArgs &a, const Place &p, const float *lds, F done) {
    constexpr int kEach = WHOLE ? 1 : E, kStride = kPlane<THREADS>;
    const int wide = WHOLE ? a.P / E : a.P;                      // values of a group in a row
    const int per = wide * a.slots, all = a.U * a.Gs;
    __syncthreads();
    const int lane = p.thread & (a.team - 1), teams = THREADS / a.team;
    for (int q0 = 0; q0 < all; q0 += teams) {
        const int q = q0 + p.thread / a.team;
        float s[K] = {};
        if (q < all) {
            const int unit = q / a.Gs, c0 = (q - unit * a.Gs) * wide, base = unit * a.A;
            for (int i = lane; i < per; i += a.team) {
                const int slot = wide == 1 ? i : static_cast<int>(__umulhi(static_cast<uint32_t>(i), a.wide_inverse));
                const int c = c0 + i - slot * wide;
                const int at = base + slot * a.L + c / kEach + c % kEach * kStride;
#pragma unroll
                for (int k = 0; k < K; ++k) s[k] += lds[k * kEach * kStride + at];
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) s[k] = group_sum_rt(s[k], a.team);
        if (q < all && lane == 0) done(q, s);
    }
    __syncthreads();
}

template <int K, int E, bool WHOLE, int THREADS, typename F>
__device__ __forceinline__ void join_groups(const GroupArgs &a, const Place &p, float *lds, const float (&v)[K][WHOLE ? 1 : E],
                                            F done) {
    constexpr int kEach = WHOLE ? 1 : E, kStride = kPlane<THREADS>;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < kEach; ++e) lds[(k * kEach + e) * kStride + p.thread] = v[k][e];
    join_lds<K, E, WHOLE, THREADS>(a, p, lds, done);
}

// The same for values that `add(e, values)` adds up: for what is rarely done, in few
// registers.  CALLS: 1, for all of a lane's channels at once (WHOLE), or E, one after the
// other, as the lanes that do it ordinarily add them.
template <int K, int CALLS, int E, bool WHOLE, int THREADS, typename V, typename F>
__device__ __forceinline__ void join_rarely(const GroupArgs &a, const Place &p, float *lds, V add, F done) {
    constexpr int kStride = kPlane<THREADS>;
    static_assert(CALLS == E || (WHOLE && CALLS == 1));
    float v[K] = {};
#pragma unroll 1
    for (int e = 0; e < CALLS; ++e) {
        add(e, v);
        if constexpr (!WHOLE)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                lds[(k * E + e) * kStride + p.thread] = v[k];
                v[k] = 0.0f;
            }
    }
    if constexpr (WHOLE)
#pragma unroll
        for (int k = 0; k < K; ++k) lds[k * kStride + p.thread] = v[k];
    join_lds<K, E, WHOLE, THREADS>(a, p, lds, done);
}

// What no group's values are (a computed NaN has another payload).
constexpr uint64_t kUnknown = ~uint64_t{0};

// A workgroup's rows: all of its samples' (held), or a member's share (shared).
struct Rows {
    int64_t n, first, count;     // sample; rows
    __device__ __forceinline__ Rows(const GroupArgs &a, int64_t sample, int member, bool shared)
        : n(sample), first(shared ? static_cast<int64_t>(member) * a.member_rows : 0),
          count(shared ? min(a.S - first, static_cast<int64_t>(a.member_rows)) : a.S) {}
};

// A workgroup's slab, its first unit of work and the way to the next: held, every so
// many samples of a slab; shared, one member of one unit, the members of a unit next to
// each other in the grid's order.
template <bool SHARED>
struct Turn {
    int slab, member;
    int64_t block, step;
    __device__ __forceinline__ explicit Turn(const GroupArgs &a) {
        // (divisions leave vector registers: what follows from them is to be scalar)
        const auto scalar = [](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v))); };
        const uint32_t slabs = a.slabs;
        if constexpr (SHARED) {
            const uint32_t members = a.members, unit = scalar(blockIdx.x / members), at = scalar(unit / slabs);
            member = static_cast<int>(blockIdx.x - unit * members);
            slab = static_cast<int>(unit - at * slabs);
            block = at;
            step = a.blocks;
        } else {
            const uint32_t at = scalar(blockIdx.x / slabs);
            member = 0;
            slab = static_cast<int>(blockIdx.x - at * slabs);
            block = at;
            step = scalar(gridDim.x / slabs);
        }
    }
};

// Publishes a group's two values (on one lane of the workgroup).
__device__ __forceinline__ void publish(uint64_t *to, float x, float y) {
    uint64_t v = static_cast<uint64_t>(__float_as_uint(y)) << 32 | __float_as_uint(x);
    if (v == kUnknown) v = 0x7fc000007fc00000u;
    __hip_atomic_store(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// All members' values of the unit's groups into LDS (known[member, group]; the
// workgroup's own are published already), and `missing(member)` -- run by the whole
// workgroup, which then has its values there too -- for those that do not appear.
template <int THREADS, typename F>
__device__ __forceinline__ void collect(const GroupArgs &a, uint64_t *unit, float2 *known, int *s_late, F missing) {
    if (threadIdx.x == 0) *s_late = 0;
    __syncthreads();
    const int all = a.members * a.Gs;
    constexpr int kAtOnce = 4;
    bool late = false;
    for (int i0 = threadIdx.x; i0 < all; i0 += kAtOnce * THREADS) {
        uint64_t v[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) v[j] = i0 + j * THREADS < all ? kUnknown : 0;
        for (int t = 0; t < a.polls; ++t) {
            bool known_all = true;
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j)
                if (v[j] == kUnknown) v[j] = __hip_atomic_load(unit + i0 + j * THREADS, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) known_all = known_all && v[j] != kUnknown;
            if (known_all) break;
            __builtin_amdgcn_s_sleep(1);
        }
        // (kUnknown as it is: what a member computes in its place is none)
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            if (i0 + j * THREADS >= all) continue;
            late = late || v[j] == kUnknown;
            known[i0 + j * THREADS] = make_float2(__uint_as_float(static_cast<uint32_t>(v[j])), __uint_as_float(static_cast<uint32_t>(v[j] >> 32)));
        }
    }
    if (late) *s_late = 1;
    __syncthreads();
    if (*s_late == 0) return;
    for (int m = 0; m < a.members; ++m) {
        bool gone = false;
        for (int g = 0; g < a.Gs; ++g)
            gone = gone || (__float_as_uint(known[m * a.Gs + g].x) == ~0u && __float_as_uint(known[m * a.Gs + g].y) == ~0u);
        __syncthreads();
        if (gone) missing(m);
        __syncthreads();
    }
}

// Sums of a lane's values, by group where a piece is of one.
template <int T, int W, bool WHOLE>
__device__ __forceinline__ void add_piece(const Piece<T, W> &x, float (&v)[WHOLE ? 1 : Piece<T, W>::kElems]) {
#pragma unroll
    for (int e = 0; e < Piece<T, W>::kElems; ++e) v[WHOLE ? 0 : e] += x[e];
}

template <int T, int W, bool WHOLE>
__device__ __forceinline__ void add_squares(const Piece<T, W> &x, const float (&mean)[WHOLE ? 1 : Piece<T, W>::kElems],
                                            float (&v)[WHOLE ? 1 : Piece<T, W>::kElems]) {
#pragma unroll
    for (int e = 0; e < Piece<T, W>::kElems; ++e) {
        const float d = x[e] - mean[WHOLE ? 0 : e];
        v[WHOLE ? 0 : e] = fmaf(d, d, v[WHOLE ? 0 : e]);
    }
}

// LDS of the held and shared forms' workgroup, in floats: values to be joined, two a
// group, two a member's group (shared), and two a channel.
__host__ __device__ inline int held_floats(int threads, int values, int groups, int known, int channels) {
    return (threads + 8) * values + 2 * groups + 2 * known + 4 + 2 * channels;
}

// Waves a SIMD that the held form is compiled for: registers for the pieces, and a
// second workgroup a CU (a third, of 256 threads) to load while one computes.
constexpr int held_waves(int threads) { return threads == 512 ? 4 : threads == 256 ? 3 : 2; }

template <int T, int W, bool WHOLE, int THREADS, int R, bool SHARED>
__global__ __launch_bounds__(THREADS, held_waves(THREADS)) void ple_group_forward_kernel(GroupArgs a) {
    constexpr int E = Piece<T, W>::kElems, kEach = WHOLE ? 1 : E;
    extern __shared__ float4 s_all[];
    float *const s_lds = reinterpret_cast<float *>(s_all);
    float *const s_mean = s_lds + kPlane<THREADS> * kEach, *const s_rho = s_mean + a.U * a.Gs;
    float2 *const s_known = reinterpret_cast<float2 *>(s_rho + a.U * a.Gs);
    int *const s_late = reinterpret_cast<int *>(s_known + a.members * a.Gs);
    float *const s_params = reinterpret_cast<float *>(s_late + 4);
    const Place here(a);
    const Turn<SHARED> turn(a);
    const int slab = turn.slab, member = turn.member;
    stage_params<THREADS>(a, slab, s_params);
    const Groups<E, WHOLE> there(a, here.lane * E);
    for (int64_t blk = turn.block; blk < a.blocks; blk += turn.step) {
        const int64_t first_n = SHARED ? blk : blk * a.U;
        const int act = unhoisted(a.act);
        const Place p = here.again();
        const Groups<E, WHOLE> groups = there.again();
        const int own = !SHARED && p.on ? p.unit * a.Gs : 0;         // the sample's groups in LDS
        const float *const own_params = s_params + (p.on ? p.lane * E : 0);
        const uint32_t at = static_cast<uint32_t>((((SHARED ? 0 : p.unit * a.S) + p.slot) * a.C + p.lane * E) * elem_bytes(T));
        const Rows rows(a, SHARED ? first_n : first_n + p.unit, member, SHARED);
        // byte offsets: the workgroup's rows (the same for all lanes), the lane's place in them
        const int64_t base = ((first_n * a.S + rows.first) * a.C + slab * a.Cs) * elem_bytes(T);
        const int64_t step = static_cast<int64_t>(a.slots) * a.C * elem_bytes(T);
        const char *const px = static_cast<const char *>(a.x) + base;
        char *const py = static_cast<char *>(a.y) + base;
        const int count = p.on && rows.n < a.N ? static_cast<int>(rows.count) - p.slot : 0;
        const auto has = [&](int k) { return k * a.slots < count; };
        Piece<T, W> x[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            x[k].clear();
            if (has(k)) x[k].load_at(px + k * step + at);
        }
        float v[1][kEach] = {};
#pragma unroll
        for (int k = 0; k < R; ++k) {
            x[k].keep();
            add_piece<T, W, WHOLE>(x[k], v[0]);
        }
        const float inv = SHARED ? a.share.inverse(member) : a.inv;
        join_groups<1, E, WHOLE, THREADS>(a, p, s_lds, v, [&](int q, const float (&s)[1]) {
            s_rho[q] = s[0];
            s_mean[q] = s[0] * inv;
        });
        float mean[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            mean[e] = s_mean[own + groups.of(e)];
            v[0][e] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            x[k].keep();
            __builtin_amdgcn_sched_barrier(0);
            if (has(k)) add_squares<T, W, WHOLE>(x[k], mean, v[0]);
        }
        if constexpr (!SHARED) {
            join_groups<1, E, WHOLE, THREADS>(a, p, s_lds, v, [&](int q, const float (&s)[1]) {
                const float rho = rsqrtf(s[0] * a.inv + a.eps);
                s_rho[q] = rho;
                const int u = q / a.Gs;
                const int64_t sample = first_n + u;
                if (sample < a.N) a.stats[sample * a.G + slab * a.Gs + (q - u * a.Gs)] = make_float2(s_mean[q], rho);
            });
        } else {
            uint64_t *const unit = a.exchange + (rows.n * a.slabs + slab) * a.members * a.Gs;
            join_groups<1, E, WHOLE, THREADS>(a, p, s_lds, v, [&](int q, const float (&s)[1]) {
                publish(unit + member * a.Gs + q, s_rho[q], s[0]);
            });
            collect<THREADS>(a, unit, s_known, s_late, [&](int m) {
                // the other member's rows
                const Rows other(a, rows.n, m, true);
                const char *const po = px + (other.first - rows.first) * a.C * elem_bytes(T) + at;
                const int there = p.on ? static_cast<int>(other.count) - p.slot : 0;
                const float share = a.share.inverse(m);
                constexpr int kCalls = WHOLE ? 1 : E;
                join_rarely<1, kCalls, E, WHOLE, THREADS>(a, p, s_lds, [&](int e0, float (&t)[1]) {
                    for (int k = 0; k * a.slots < there; ++k)
                        for (int e = e0; e < e0 + E / kCalls; ++e) t[0] += load_grad<T>(po + k * step, e);
                }, [&](int q, const float (&s)[1]) {
                    s_rho[q] = s[0];
                    s_mean[q] = s[0] * share;
                });
                join_rarely<1, kCalls, E, WHOLE, THREADS>(a, p, s_lds, [&](int e0, float (&t)[1]) {
                    const float mu = s_mean[own + groups.of(e0)];
                    for (int k = 0; k * a.slots < there; ++k)
                        for (int e = e0; e < e0 + E / kCalls; ++e) {
                            const float d = load_grad<T>(po + k * step, e) - mu;
                            t[0] = fmaf(d, d, t[0]);
                        }
                }, [&](int q, const float (&s)[1]) { s_known[m * a.Gs + q] = make_float2(s_rho[q], s[0]); });
            });
            // the unit's mean, and its squares about it: the members' own, and their means' distance
            const int lane = p.thread & (a.team - 1);
            for (int q0 = 0; q0 < a.Gs; q0 += THREADS / a.team) {
                const int q = q0 + p.thread / a.team;
                float t = 0.0f;
                if (q < a.Gs)
                    for (int m = lane; m < a.members; m += a.team) t += s_known[m * a.Gs + q].x;
                const float mu = group_sum_rt(t, a.team) * a.inv;
                t = 0.0f;
                if (q < a.Gs)
                    for (int m = lane; m < a.members; m += a.team) {
                        const float2 s = s_known[m * a.Gs + q];
                        t += s.y + a.share.distance(s.x, m, mu);
                    }
                t = group_sum_rt(t, a.team);
                if (q < a.Gs && lane == 0) {
                    const float rho = rsqrtf(t * a.inv + a.eps);
                    s_mean[q] = mu;
                    s_rho[q] = rho;
                    if (member == 0) a.stats[rows.n * a.G + slab * a.Gs + q] = make_float2(mu, rho);
                }
            }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kEach; ++e) mean[e] = s_mean[own + groups.of(e)];
        }
        float scale[E], bias[E];
        staged(own_params, scale);
        staged(own_params + a.Cs, bias);
#pragma unroll
        for (int e = 0; e < E; ++e) scale[e] *= s_rho[own + groups.of(e)];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            x[k].keep();
            __builtin_amdgcn_sched_barrier(0);
            if (has(k)) {
                float z[E];
#pragma unroll
                for (int e = 0; e < E; ++e) z[e] = fmaf(x[k][e] - mean[WHOLE ? 0 : e], scale[e], bias[e]);
                activate(z, act);
                store_piece<T, W>(py + k * step + at, 0, z);
            }
        }
        if constexpr (SHARED) break;
        __syncthreads();             // (s_mean and s_rho are read before the next samples')
    }
}

// The parameters' gradient sums of a workgroup's lanes, by channel: a partial.
template <int E, int THREADS>
__device__ __forceinline__ void leave_sums(const GroupArgs &a, const Place &p, float *lds, const float (&v)[2][E], int slab,
                                           int64_t part) {
    constexpr int kStride = kPlane<THREADS>;
    const int rows = a.U * a.slots;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; ++e) lds[e * kStride + p.thread] = v[k][e];
        __syncthreads();
        for (int c = p.thread; c < a.Cs; c += THREADS) {
            float s = 0.0f;
            for (int i = 0; i < rows; ++i) s += lds[c % E * kStride + i * a.L + c / E];
            a.partial[(part * 2 + k) * a.C + slab * a.Cs + c] = s;
        }
    }
}

// A lane's channels before the activation: z = (x - mean) scale + bias, in the order and with
// the roundings of the forward, so that a relu's gradient passes where its output is above 0.
template <int E, bool WHOLE>
struct Affine {
    float scale[E], bias[E], mean[WHOLE ? 1 : E];
    __device__ __forceinline__ Affine(const float *weight, const float *biases, const float2 *stats, const Groups<E, WHOLE> &groups) {
        staged(weight, scale);
        staged(biases, bias);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float2 st = stats[groups.of(e)];
            scale[e] *= st.y;
            mean[WHOLE ? 0 : e] = st.x;
        }
    }
};

// x - mean of a piece.  Pieces of 32-bit values hold it in the place of x (centre), which
// saves the registers of the means.
template <int T, int W, int E, bool WHOLE>
__device__ __forceinline__ void centre(Piece<T, W> &x, const Affine<E, WHOLE> &f) {
    if constexpr (T == PLE_DTYPE_F32)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x.w[e] = __float_as_uint(x[e] - f.mean[WHOLE ? 0 : e]);
            asm volatile("" : "+v"(x.w[e]));         // (here, and not where it is used)
        }
}

template <int T, int W, int E, bool WHOLE>
__device__ __forceinline__ void distances(const Piece<T, W> &x, const Affine<E, WHOLE> &f, float (&d)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) d[e] = T == PLE_DTYPE_F32 ? x[e] : x[e] - f.mean[WHOLE ? 0 : e];
}

// A piece's gradient before the activation, from its distances.
template <int T, int W, int E, bool WHOLE>
__device__ __forceinline__ void piece_grad(int act, const float (&d)[E], const Piece<T, W> &g, const Affine<E, WHOLE> &f,
                                           float (&dz)[E]) {
#pragma clang fp contract(off)
#pragma unroll
    for (int e = 0; e < E; ++e) dz[e] = fmaf(d[e], f.scale[e], f.bias[e]);
    slopes(dz, act);
#pragma unroll
    for (int e = 0; e < E; ++e) dz[e] *= g[e];
}

// Sums of dz and dz (x - mean) of a lane's channels -> of dz and dz xh.  (Of dz x, less mean
// times the sum of dz, they lost what the mean is larger than the deviation.)
template <int E, bool WHOLE>
__device__ __forceinline__ void standard_sums(const float2 *stats, const Groups<E, WHOLE> &groups, float (&sum)[2][E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) sum[1][e] *= stats[groups.of(e)].y;
}

// ... weighted, by group where a piece is of one.
template <int E, bool WHOLE>
__device__ __forceinline__ void weigh_sums(const float *weight, const float (&sum)[2][E], float (&v)[2][WHOLE ? 1 : E]) {
    float w[E];
    staged(weight, w);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < E; ++e) v[j][WHOLE ? 0 : e] = fmaf(sum[j][e], w[e], v[j][WHOLE ? 0 : e]);
}

// Waves a SIMD that the backward is compiled for (its largest 32-bit pieces just fit four:
// 8192 x 64 x 96 in groups of 3 119 us, with three 131).
constexpr int backward_waves(int type, int words, bool shared) {
    return shared ? 3 : type == PLE_DTYPE_F32 && words == 4 ? 4 : 2;
}

template <int T, int W, bool WHOLE, int THREADS, int R, bool SHARED>
__global__ __launch_bounds__(THREADS, backward_waves(T, W, SHARED)) void ple_group_backward_kernel(GroupArgs a) {
    constexpr int E = Piece<T, W>::kElems, kEach = WHOLE ? 1 : E, kValues = 2 * kEach > E ? 2 * kEach : E;
    extern __shared__ float4 s_all[];
    float *const s_lds = reinterpret_cast<float *>(s_all);
    float *const s_m1 = s_lds + kPlane<THREADS> * kValues, *const s_m2 = s_m1 + a.U * a.Gs;
    float2 *const s_known = reinterpret_cast<float2 *>(s_m2 + a.U * a.Gs);
    int *const s_late = reinterpret_cast<int *>(s_known + a.members * a.Gs);
    float *const s_params = reinterpret_cast<float *>(s_late + 4);
    const Place here(a);
    const Turn<SHARED> turn(a);
    const int slab = turn.slab, member = turn.member;
    stage_params<THREADS>(a, slab, s_params);
    __syncthreads();
    const Groups<E, WHOLE> there(a, here.lane * E);
    float all[2][E] = {};
    for (int64_t blk = turn.block; blk < a.blocks; blk += turn.step) {
        const int64_t first_n = SHARED ? blk : blk * a.U;
        const int act = unhoisted(a.act);
        const Place p = here.again();
        const Groups<E, WHOLE> groups = there.again();
        const int own = !SHARED && p.on ? p.unit * a.Gs : 0;         // the sample's groups in LDS
        const float *const own_params = s_params + (p.on ? p.lane * E : 0);
        const uint32_t at = static_cast<uint32_t>((((SHARED ? 0 : p.unit * a.S) + p.slot) * a.C + p.lane * E) * elem_bytes(T));
        const Rows rows(a, SHARED ? first_n : first_n + p.unit, member, SHARED);
        const int64_t base = ((first_n * a.S + rows.first) * a.C + slab * a.Cs) * elem_bytes(T);
        const int64_t step = static_cast<int64_t>(a.slots) * a.C * elem_bytes(T);
        const char *const px = static_cast<const char *>(a.x) + base;
        const char *const pg = static_cast<const char *>(a.g) + base;
        char *const py = static_cast<char *>(a.y) + base;
        const int count = p.on && rows.n < a.N ? static_cast<int>(rows.count) - p.slot : 0;
        const auto has = [&](int k) { return k * a.slots < count; };
        // (lanes without rows read the statistics of the last sample's)
        const float2 *const stats = a.stats + (SHARED ? first_n : min(p.on ? rows.n : first_n, a.N - 1)) * a.G + slab * a.Gs;
        Piece<T, W> x[R], g[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            x[k].clear();
            g[k].clear();
            if (has(k)) {
                x[k].load_at(px + k * step + at);
                g[k].load_at(pg + k * step + at);
            }
        }
        // dz is kept until the groups' sums are known (8 x 65536 x 256 bf16 in groups of 8,
        // when this was chosen: 233 us, computed again 277), where three workgroups have the
        // registers for it (16 x 4096 x 320 in groups of 10: 50 us either way, kept in part in
        // scratch memory)
        constexpr bool kKept = WHOLE || !SHARED || E < 8;
        float sum[2][E] = {}, grad[kKept ? R : 1][E];
        {
            const Affine<E, WHOLE> f(own_params, own_params + a.Cs, stats, groups);
#pragma unroll
            for (int k = 0; k < R; ++k) centre(x[k], f);
#pragma unroll
            for (int k = 0; k < R; ++k) {
                x[k].keep();
                g[k].keep();
                __builtin_amdgcn_sched_barrier(0);
                // (a row that is not there has a gradient of 0)
                float d[E];
                float (&dz)[E] = grad[kKept ? k : 0];
                distances(x[k], f, d);
                piece_grad<T, W>(act, d, g[k], f, dz);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    sum[0][e] += dz[e];
                    sum[1][e] = fmaf(dz[e], d[e], sum[1][e]);
                    // (here, and not where the sums are used: the terms would all be held)
                    asm volatile("" : "+v"(sum[0][e]), "+v"(sum[1][e]), "+v"(dz[e]));
                }
            }
        }
        standard_sums<E, WHOLE>(stats, groups, sum);
        float v[2][kEach] = {};
        weigh_sums<E, WHOLE>(own_params, sum, v);
        if constexpr (!SHARED) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < E; ++e) all[j][e] += sum[j][e];
            if (!a.y) continue;
            join_groups<2, E, WHOLE, THREADS>(a, p, s_lds, v, [&](int q, const float (&s)[2]) {
                s_m1[q] = s[0] * a.inv;
                s_m2[q] = s[1] * a.inv;
            });
        } else {
            uint64_t *const unit = a.exchange + (rows.n * a.slabs + slab) * a.members * a.Gs;
            if (a.y)
                join_groups<2, E, WHOLE, THREADS>(a, p, s_lds, v, [&](int q, const float (&s)[2]) {
                    publish(unit + member * a.Gs + q, s[0], s[1]);
                });
            // (while the others' are on their way)
            if (a.partial) leave_sums<E, THREADS>(a, p, s_lds, sum, slab, blk * a.members + member);
            if (!a.y) break;
            collect<THREADS>(a, unit, s_known, s_late, [&](int m) {
                const Rows other(a, rows.n, m, true);
                const int64_t away = (other.first - rows.first) * a.C * elem_bytes(T) + at;
                const int there = p.on ? static_cast<int>(other.count) - p.slot : 0;
                join_rarely<2, E, E, WHOLE, THREADS>(a, p, s_lds, [&](int e, float (&v)[2]) {
#pragma clang fp contract(off)
                    const float2 st = stats[groups.of(e)];
                    const float w = own_params[e], scale = w * st.y, bias = own_params[a.Cs + e];
                    float t[2] = {};
                    for (int k = 0; k * a.slots < there; ++k) {
                        const float d = load_grad<T>(px + away + k * step, e) - st.x;
                        float dz[1] = {fmaf(d, scale, bias)};
                        slopes(dz, act);
                        dz[0] *= load_grad<T>(pg + away + k * step, e);
                        t[0] += dz[0];
                        t[1] = fmaf(dz[0], d, t[1]);
                    }
                    v[0] = fmaf(t[0], w, v[0]);
                    v[1] = fmaf(t[1] * st.y, w, v[1]);
                }, [&](int q, const float (&r)[2]) { s_known[m * a.Gs + q] = make_float2(r[0], r[1]); });
            });
            const int lane = p.thread & (a.team - 1);
            for (int q0 = 0; q0 < a.Gs; q0 += THREADS / a.team) {
                const int q = q0 + p.thread / a.team;
                float t = 0.0f, u = 0.0f;
                if (q < a.Gs)
                    for (int m = lane; m < a.members; m += a.team) {
                        t += s_known[m * a.Gs + q].x;
                        u += s_known[m * a.Gs + q].y;
                    }
                t = group_sum_rt(t, a.team);
                u = group_sum_rt(u, a.team);
                if (q < a.Gs && lane == 0) {
                    s_m1[q] = t * a.inv;
                    s_m2[q] = u * a.inv;
                }
            }
            __syncthreads();
        }
        // dx = dz scale + (x - mean) along + level
        const Affine<E, WHOLE> f(own_params, own_params + a.Cs, stats, groups);
        float along[kEach], level[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const float2 st = stats[groups.of(e)];
            const int q = own + groups.of(e);
            along[e] = -st.y * st.y * s_m2[q];
            level[e] = -st.y * s_m1[q];
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            x[k].keep();
            if constexpr (!kKept) g[k].keep();
            __builtin_amdgcn_sched_barrier(0);
            float d[E];
            float (&dz)[E] = grad[kKept ? k : 0];
            distances(x[k], f, d);
            if constexpr (!kKept) piece_grad<T, W>(act, d, g[k], f, dz);
#pragma unroll
            for (int e = 0; e < E; ++e)
                dz[e] = dz[e] * f.scale[e] + (d[e] * along[WHOLE ? 0 : e] + level[WHOLE ? 0 : e]);
            if (has(k)) store_piece<T, W>(py + k * step + at, 0, dz);
        }
        if constexpr (SHARED) break;
        __syncthreads();
    }
    if constexpr (!SHARED)
        if (a.partial) leave_sums<E, THREADS>(a, here.again(), s_lds, all, slab, turn.block);
}

// Clears the words that members exchange.
__global__ __launch_bounds__(kBlock) void ple_group_unknown_kernel(uint64_t *p, int64_t n) {
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * kBlock)
        p[i] = kUnknown;
}

// ---------------------------------------------------------------------------
// split form
// ---------------------------------------------------------------------------

constexpr int kSplitRows = 8;        // rows a lane holds of a piece

// A workgroup's piece of a sample: rows [first, first + slots * kSplitRows) of the
// channels of its slab (the last slab may be narrower).
struct Split {
    int slab, slot, lane;
    int64_t n, row;
    int piece, c0;
    bool on;
    __device__ __forceinline__ Split(const GroupArgs &a, int E, int64_t blk) : Split(a, E, blk, static_cast<int>(threadIdx.x)) {}
    __host__ __device__ __forceinline__ Split(const GroupArgs &a, int E, int64_t blk, int thread) {
        slot = thread / a.L;
        lane = thread - slot * a.L;
        const int64_t u = blk / a.slabs;
        slab = static_cast<int>(blk - u * a.slabs);
        n = u / a.pieces;
        piece = static_cast<int>(u - n * a.pieces);
        row = static_cast<int64_t>(piece) * a.slots * kSplitRows + slot;
        c0 = slab * a.Cs + lane * E;
        on = slot < a.slots && c0 < a.C;
    }
};

// A lane's channels of the split form: their parameters and groups.
template <int E>
struct SplitChannels {
    float w[E], b[E];
    Groups<E, false> groups;
    int last;
    __device__ __forceinline__ SplitChannels(const GroupArgs &a, int c0) : groups(a, c0), last(a.G - 1) {
        load_params(a, a.weight, first_param(a, c0), 1.0f, w);
        load_params(a, a.bias, first_param(a, c0), 0.0f, b);
    }
    // Where a lane reads its E parameters (the last slab may be narrower: its lanes without
    // channels read the last ones).
    __host__ __device__ static __forceinline__ int first_param(const GroupArgs &a, int c0) { return min(c0, a.C - E); }
    __device__ __forceinline__ int of(int e) const { return min(groups.of(e), last); }
};

// Sums over the workgroup's row slots of a value a channel, to `done(channel, sum)`.
template <int E, typename F>
__device__ __forceinline__ void join_slots(const GroupArgs &a, const Split &p, float *lds, const float (&v)[E], F done) {
    if (p.slot < a.slots)
#pragma unroll
        for (int e = 0; e < E; ++e) lds[p.slot * a.Cs + p.lane * E + e] = v[e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.Cs; c += kBlock) {
        float s = 0.0f;
        for (int i = 0; i < a.slots; ++i) s += lds[i * a.Cs + c];
        done(c, s);
    }
    __syncthreads();
}

// Sum and squares about the mean of a piece's channels.
template <int T, int W>
__global__ __launch_bounds__(kBlock) void ple_group_sums_kernel(GroupArgs a) {
    constexpr int E = Piece<T, W>::kElems;
    extern __shared__ float s_lds[];
    float *const s_sum = s_lds + a.slots * a.Cs;
    for (int64_t blk = blockIdx.x; blk < a.blocks; blk += gridDim.x) {
        const Split p(a, E, blk);
        Piece<T, W> x[kSplitRows];
#pragma unroll
        for (int k = 0; k < kSplitRows; ++k) {
            x[k].clear();
            if (p.on && p.row + k * a.slots < a.S) x[k].load(a.x, (p.n * a.S + p.row + k * a.slots) * a.C + p.c0);
        }
        const float inv = a.share.inverse(p.piece);
        float v[E] = {};
#pragma unroll
        for (int k = 0; k < kSplitRows; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] += x[k][e];
        join_slots(a, p, s_lds, v, [&](int c, float s) { s_sum[c] = s; });
        float mean[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            mean[e] = p.slot < a.slots ? s_sum[p.lane * E + e] * inv : 0.0f;
            v[e] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < kSplitRows; ++k)
            if (p.row + k * a.slots < a.S)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = x[k][e] - mean[e];
                    v[e] += d * d;
                }
        join_slots(a, p, s_lds, v, [&](int c, float s) {
            const int at = p.slab * a.Cs + c;
            if (at < a.C) a.sums[(p.n * a.pieces + p.piece) * a.C + at] = make_float2(s_sum[c], s);
        });
    }
}

// Sum over the workgroup, to all of its threads.
__device__ __forceinline__ float block_sum(float v, float *lds) {
    v = group_sum<kWave>(v);
    __syncthreads();
    if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kWavesPerBlock; ++i) s += lds[i];
    return s;
}

// Folds kFold pieces into one, channel by channel: the sums and the squares about the
// mean (CENTRED), or two sums.  (A sample's groups are too few workgroups to read many
// pieces: 1 x 60000 x 960 bf16 in 10 groups, 1875 pieces, fold and join of the backward
// 19 us, the join alone 273.)
constexpr int kFold = 32;

template <bool CENTRED>
__global__ __launch_bounds__(kBlock) void ple_group_fold_kernel(GroupArgs a) {
    const int64_t all = a.N * a.folded * a.C;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x; i < all; i += static_cast<int64_t>(gridDim.x) * kBlock) {
        const int64_t t = i / a.C, n = t / a.folded;
        const int c = static_cast<int>(i - t * a.C), first = static_cast<int>(t - n * a.folded) * kFold;
        const int last = min(a.pieces, first + kFold);
        const float2 *const p = a.sums + n * a.pieces * a.C + c;
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll 8
        for (int j = first; j < last; ++j) {
            const float2 v = p[static_cast<int64_t>(j) * a.C];
            s.x += v.x;
            s.y += v.y;
        }
        if constexpr (CENTRED) {
            const float mean = s.x * a.fold.inverse(first / kFold);
            float t = 0.0f;
#pragma unroll 8
            for (int j = first; j < last; ++j) t += a.share.distance(p[static_cast<int64_t>(j) * a.C].x, j, mean);
            s.y += t;
        }
        a.folds[i] = s;
    }
}

// What the joins read after a fold.
inline GroupArgs folded_args(GroupArgs a) {
    if (a.folded > 0) {
        a.sums = a.folds;
        a.pieces = a.folded;
        a.share = a.fold;
    }
    return a;
}

// Mean and factor of a sample's group from its pieces: the squares about a piece's
// mean, and the mean's own distance.
__global__ __launch_bounds__(kBlock) void ple_group_stats_kernel(GroupArgs a) {
    __shared__ float s_lds[kWavesPerBlock];
    for (int64_t ng = blockIdx.x; ng < a.N * a.G; ng += gridDim.x) {
        const int64_t n = ng / a.G;
        const int g = static_cast<int>(ng - n * a.G);
        const float2 *sums = a.sums + n * a.pieces * a.C + g * a.P;
        const int64_t all = static_cast<int64_t>(a.pieces) * a.P;
        float t = 0.0f;
        for (int64_t i = threadIdx.x; i < all; i += kBlock) t += sums[i / a.P * a.C + i % a.P].x;
        const float mean = block_sum(t, s_lds) * a.inv;
        t = 0.0f;
        for (int64_t i = threadIdx.x; i < all; i += kBlock) {
            const int64_t piece = i / a.P;
            const float2 s = sums[piece * a.C + i % a.P];
            t += s.y + a.share.distance(s.x, static_cast<int>(piece), mean);
        }
        t = block_sum(t, s_lds);
        if (threadIdx.x == 0) a.stats[ng] = make_float2(mean, rsqrtf(t * a.inv + a.eps));
    }
}

template <int T, int W>
__global__ __launch_bounds__(kBlock) void ple_group_apply_kernel(GroupArgs a) {
    constexpr int E = Piece<T, W>::kElems;
    for (int64_t blk = blockIdx.x; blk < a.blocks; blk += gridDim.x) {
        const Split p(a, E, blk);
        if (!p.on) continue;
        const SplitChannels<E> ch(a, p.c0);
        float mean[E], scale[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float2 s = a.stats[p.n * a.G + ch.of(e)];
            mean[e] = s.x;
            scale[e] = s.y * ch.w[e];
        }
        Piece<T, W> x[kSplitRows];
#pragma unroll
        for (int k = 0; k < kSplitRows; ++k)
            if (p.row + k * a.slots < a.S) x[k].load(a.x, (p.n * a.S + p.row + k * a.slots) * a.C + p.c0);
#pragma unroll
        for (int k = 0; k < kSplitRows; ++k)
            if (p.row + k * a.slots < a.S) {
                float z[E];
#pragma unroll
                for (int e = 0; e < E; ++e) z[e] = fmaf(x[k][e] - mean[e], scale[e], ch.b[e]);
                activate(z, a.act);
                store_piece<T, W>(a.y, (p.n * a.S + p.row + k * a.slots) * a.C + p.c0, z);
            }
    }
}

// Sums of dz and dz xh of a piece's channels.
template <int T, int W>
__global__ __launch_bounds__(kBlock) void ple_group_backward_sums_kernel(GroupArgs a) {
    constexpr int E = Piece<T, W>::kElems;
    extern __shared__ float s_lds[];
    float *const s_sum = s_lds + a.slots * a.Cs;
    for (int64_t blk = blockIdx.x; blk < a.blocks; blk += gridDim.x) {
        const Split p(a, E, blk);
        const SplitChannels<E> ch(a, p.c0);
        float v[E] = {}, u[E] = {};
        if (p.on) {
            float2 st[E];
#pragma unroll
            for (int e = 0; e < E; ++e) st[e] = a.stats[p.n * a.G + ch.of(e)];
            Piece<T, W> x[kSplitRows], g[kSplitRows];
#pragma unroll
            for (int k = 0; k < kSplitRows; ++k)
                if (p.row + k * a.slots < a.S) {
                    const int64_t at = (p.n * a.S + p.row + k * a.slots) * a.C + p.c0;
                    x[k].load(a.x, at);
                    g[k].load(a.g, at);
                }
#pragma unroll
            for (int k = 0; k < kSplitRows; ++k)
                if (p.row + k * a.slots < a.S) {
                    float xh[E], dz[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float d = x[k][e] - st[e].x;
                        xh[e] = d * st[e].y;
                        dz[e] = fmaf(d, st[e].y * ch.w[e], ch.b[e]);     // (as the forward)
                    }
                    slopes(dz, a.act);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float d = dz[e] * g[k][e];
                        v[e] += d;
                        u[e] += d * xh[e];
                    }
                }
        }
        join_slots(a, p, s_lds, v, [&](int c, float s) { s_sum[c] = s; });
        join_slots(a, p, s_lds, u, [&](int c, float s) {
            const int at = p.slab * a.Cs + c;
            if (at < a.C) a.sums[(p.n * a.pieces + p.piece) * a.C + at] = make_float2(s_sum[c], s);
        });
    }
}

// A sample's group: its channels' sums over the pieces, and the means of g and g xh.
__global__ __launch_bounds__(kBlock) void ple_group_backward_join_kernel(GroupArgs a) {
    __shared__ float s_lds[2 * kBlock];
    const int wide = min(a.P, kBlock), slots = kBlock / wide;
    const int slot = threadIdx.x / wide, lane = threadIdx.x - slot * wide;
    for (int64_t ng = blockIdx.x; ng < a.N * a.G; ng += gridDim.x) {
        const int64_t n = ng / a.G;
        const int g = static_cast<int>(ng - n * a.G);
        float m1 = 0.0f, m2 = 0.0f;
        for (int c1 = 0; c1 < a.P; c1 += wide) {
            const int c = g * a.P + c1 + lane;
            const bool on = slot < slots && c1 + lane < a.P;
            float2 s = make_float2(0.0f, 0.0f);
            if (on)
                for (int i = slot; i < a.pieces; i += slots) {
                    const float2 t = a.sums[(n * a.pieces + i) * a.C + c];
                    s.x += t.x;
                    s.y += t.y;
                }
            __syncthreads();
            s_lds[threadIdx.x] = s.x;
            s_lds[kBlock + threadIdx.x] = s.y;
            __syncthreads();
            if (on && slot == 0) {
                for (int i = 1; i < slots; ++i) {
                    s.x += s_lds[i * wide + lane];
                    s.y += s_lds[kBlock + i * wide + lane];
                }
                a.channels[n * a.C + c] = s;
                const float w = a.weight ? load_any(a.weight, c, a.param_dtype) : 1.0f;
                m1 += w * s.x;
                m2 += w * s.y;
            }
        }
        m1 = block_sum(m1, s_lds);
        m2 = block_sum(m2, s_lds);
        if (threadIdx.x == 0) a.means[ng] = make_float2(m1 * a.inv, m2 * a.inv);
    }
}

template <int T, int W>
__global__ __launch_bounds__(kBlock) void ple_group_backward_apply_kernel(GroupArgs a) {
    constexpr int E = Piece<T, W>::kElems;
    for (int64_t blk = blockIdx.x; blk < a.blocks; blk += gridDim.x) {
        const Split p(a, E, blk);
        if (!p.on) continue;
        const SplitChannels<E> ch(a, p.c0);
        float2 st[E], m[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            st[e] = a.stats[p.n * a.G + ch.of(e)];
            m[e] = a.means[p.n * a.G + ch.of(e)];
        }
        Piece<T, W> x[kSplitRows], g[kSplitRows];
#pragma unroll
        for (int k = 0; k < kSplitRows; ++k)
            if (p.row + k * a.slots < a.S) {
                const int64_t at = (p.n * a.S + p.row + k * a.slots) * a.C + p.c0;
                x[k].load(a.x, at);
                g[k].load(a.g, at);
            }
#pragma unroll
        for (int k = 0; k < kSplitRows; ++k)
            if (p.row + k * a.slots < a.S) {
                float xh[E], dz[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = x[k][e] - st[e].x;
                    xh[e] = d * st[e].y;
                    dz[e] = fmaf(d, st[e].y * ch.w[e], ch.b[e]);
                }
                slopes(dz, a.act);
#pragma unroll
                for (int e = 0; e < E; ++e) dz[e] = st[e].y * (dz[e] * g[k][e] * ch.w[e] - m[e].x - xh[e] * m[e].y);
                store_piece<T, W>(a.y, (p.n * a.S + p.row + k * a.slots) * a.C + p.c0, dz);
            }
    }
}

// ---------------------------------------------------------------------------
// the parameters' gradients
// ---------------------------------------------------------------------------

struct ParamJoin {
    const float *sums;           // sum k (0: dz, 1: dz xh) of channel c of a part: sums[part * part_stride + k * sum_stride + c * step]
    void *bias, *weight;
    int64_t parts, part_stride, sum_stride;
    int step, C, param_dtype;
};

// 16 channels a workgroup, its 64 rows of lanes a part each in turn; blockIdx.y: which sum
constexpr int kParamChannels = 16, kParamThreads = 1024;

__global__ __launch_bounds__(kParamThreads) void ple_group_param_kernel(ParamJoin a) {
    constexpr int kRows = kParamThreads / kParamChannels;
    __shared__ float s_sum[kParamThreads];
    const int row = threadIdx.x / kParamChannels, c = blockIdx.x * kParamChannels + threadIdx.x % kParamChannels, k = blockIdx.y;
    float v = 0.0f;
    if (c < a.C) {
#pragma unroll 8
        for (int64_t p = row; p < a.parts; p += kRows)
            v += a.sums[p * a.part_stride + k * a.sum_stride + static_cast<int64_t>(c) * a.step];
    }
    s_sum[threadIdx.x] = v;
    __syncthreads();
    void *const out = k == 0 ? a.bias : a.weight;
    if (row == 0 && c < a.C && out) {
#pragma unroll 8
        for (int r = 1; r < kRows; ++r) v += s_sum[r * kParamChannels + threadIdx.x];
        store_any(out, c, v, a.param_dtype);
    }
}

// ---------------------------------------------------------------------------
// plans and launches
// ---------------------------------------------------------------------------

struct GroupPlan {
    int words;                   // a lane's piece: 4, 1 or 0 dwords
    int E;
    bool whole, held, shared;    // held: also where it is shared
    int threads, rows;           // held: threads and rows a lane (both compile-time)
    int L, slots, U, slabs, Cs, Gs, team, pieces;
    int members, member_rows, folded;
    int64_t blocks, parts;
    size_t lds, o_exchange, o_channels, o_means, o_folds, bytes;
};

// The widest piece that divides a row's slab and its address.
int piece_words(int dtype, int64_t channels, bool aligned16, bool aligned4) {
    const int64_t bytes = channels * elem_bytes(dtype);
    if (aligned16 && bytes % 16 == 0) return 4;
    if (aligned4 && bytes % 4 == 0) return 1;
    return 0;
}

int piece_elems(int dtype, int words) { return words == 0 ? 1 : (dtype == PLE_DTYPE_F32 ? words : 2 * words); }

// The workgroups and pieces a lane of the held form, for pieces of 4 dwords (narrower
// ones: four times as many of them).  The last is the shared form's, which rather has
// more members.
struct HeldShape {
    int threads, rows;
};
constexpr HeldShape kForwardShapes[] = {{64, 4}, {64, 16}, {256, 16}, {512, 16}};
constexpr HeldShape kBackwardShapes[] = {{64, 4}, {64, 8}, {256, 4}, {256, 8}};
constexpr int kShapes = 4;
constexpr int kMaxMembers = 320;         // of a unit: fewer than workgroups run at once
constexpr int kMaxKnown = 4096;          // groups of all members

constexpr int rows_of(const HeldShape &s, int words, bool shared) { return words == 4 || shared ? s.rows : 4 * s.rows; }

// The slab of gs groups as a workgroup's: false where its lanes or LDS do not fit.
bool hold(const GroupRequest &r, bool backward, int64_t gs, bool aligned16, bool aligned4, const HeldShape &shape, bool share,
          GroupPlan &p) {
    const int64_t P = r.C / r.G, Cs = gs * P;
    p.words = piece_words(r.dtype, gs < r.G ? Cs : r.C, aligned16 && (gs == r.G || r.C * elem_bytes(r.dtype) % 16 == 0),
                          aligned4 && (gs == r.G || r.C * elem_bytes(r.dtype) % 4 == 0));
    p.E = piece_elems(r.dtype, p.words);
    const int64_t L = Cs / p.E;
    if (L > shape.threads) return false;
    p.whole = p.E != 2 && P % p.E == 0;          // (with_held's kernels)
    p.threads = shape.threads;
    p.rows = rows_of(shape, p.words, share);
    p.L = static_cast<int>(L);
    p.slots = static_cast<int>(std::min<int64_t>(r.S, shape.threads / L));
    // many samples: as few lanes each as hold them, so that more of them are loaded at once
    // (65536 x 8 x 24 fp32 step: 147 us with all lanes that its rows have, 64 so)
    const int64_t fewest = (r.S + p.rows - 1) / p.rows;
    if (!share && fewest < p.slots && r.N * L * fewest >= 1024 * static_cast<int64_t>(device_cu_count())) p.slots = static_cast<int>(fewest);
    p.slabs = static_cast<int>(r.G / gs); p.Cs = static_cast<int>(Cs); p.Gs = static_cast<int>(gs);
    if (!share && static_cast<int64_t>(p.slots) * p.rows < r.S) return false;
    const int A = p.L * p.slots;
    p.U = share ? 1 : static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(p.threads / A, r.N)));
    p.blocks = (r.N + p.U - 1) / p.U;
    p.members = 0;
    if (share) {
        // as many members as hold it, or as give every CU two workgroups, of 16 KB at least
        const int64_t need = (r.S + static_cast<int64_t>(p.slots) * p.rows - 1) / (static_cast<int64_t>(p.slots) * p.rows);
        const int64_t fill = 2 * device_cu_count() / (r.N * p.slabs), most = r.S * Cs * elem_bytes(r.dtype) / 16384;
        const int64_t want = std::max(need, std::min({fill, most, static_cast<int64_t>(kMaxMembers), kMaxKnown / gs}));
        p.member_rows = static_cast<int>(((r.S + want - 1) / want + p.slots - 1) / p.slots * p.slots);
        const int64_t members = (r.S + p.member_rows - 1) / p.member_rows;
        if (members > kMaxMembers || members * gs > kMaxKnown || r.N * p.slabs * members > (1 << 22)) return false;
        p.members = static_cast<int>(members);
    }
    const int each = p.whole ? 1 : p.E, values = static_cast<int>((p.whole ? P / p.E : P) * p.slots), groups = p.U * p.Gs;
    p.team = 1;
    while (p.team < kWave && 2 * p.team * groups <= p.threads && 2 * p.team <= values) p.team *= 2;
    p.lds = 4 * static_cast<size_t>(held_floats(p.threads, backward ? std::max(2 * each, p.E) : each, groups, p.members * p.Gs, p.Cs));
    return p.lds <= kLdsMax / 2;
}

GroupPlan plan_group(const GroupRequest &r, bool backward, bool aligned16, bool aligned4) {
    GroupPlan p{};
    const HeldShape *shapes = backward ? kBackwardShapes : kForwardShapes;
    const int64_t P = r.C / r.G;
    const auto lines = [&](int64_t gs) { return gs * P * elem_bytes(r.dtype) >= 128; };
    // held: as many groups a workgroup as fit, the smallest workgroup that does; a slab's
    // part of a row is a cache line or more
    for (int64_t gs = r.G; gs >= 1 && !p.held && (gs == r.G || lines(gs)); --gs) {
        if (r.G % gs != 0) continue;
        for (int i = 0; i < kShapes && !p.held; ++i) p.held = hold(r, backward, gs, aligned16, aligned4, shapes[i], false, p);
    }
    // shared: where a sample's slab is too large for that, or there are too few for half of
    // the CUs.  The narrowest slab of whole cache lines, or the row.
    if (!p.held || (r.N * p.slabs < device_cu_count() / 2 && static_cast<int64_t>(p.Cs) * r.S * elem_bytes(r.dtype) > 65536)) {
        GroupPlan q{};
        int64_t gs = r.G;
        for (int64_t g = r.G; g >= 1; --g)
            if (r.G % g == 0 && lines(g) && g * P * elem_bytes(r.dtype) % 128 == 0) gs = g;
        if (hold(r, backward, gs, aligned16, aligned4, shapes[kShapes - 1], true, q)) {
            p = q;
            p.held = p.shared = true;
        }
    }
    if (!p.held) {
        p = GroupPlan{};
        p.words = piece_words(r.dtype, r.C, aligned16, aligned4);
        p.E = piece_elems(r.dtype, p.words);
        const int64_t lanes = (r.C + p.E - 1) / p.E;
        p.slabs = static_cast<int>((lanes + 63) / 64);
        p.L = static_cast<int>((lanes + p.slabs - 1) / p.slabs);
        p.Cs = p.L * p.E;
        p.slots = kBlock / p.L;
        p.pieces = static_cast<int>((r.S + static_cast<int64_t>(p.slots) * kSplitRows - 1) / (p.slots * kSplitRows));
        p.blocks = r.N * p.pieces * p.slabs;
        p.lds = static_cast<size_t>(p.slots + 1) * p.Cs * 4;
        p.o_channels = align_up(static_cast<size_t>(r.N) * p.pieces * r.C * 8, 256);
        p.o_means = p.o_channels + (backward ? align_up(static_cast<size_t>(r.N) * r.C * 8, 256) : 0);
        p.o_folds = p.o_means + (backward ? align_up(static_cast<size_t>(r.N) * r.G * 8, 256) : 0);
        p.folded = p.pieces > 2 * kFold ? (p.pieces + kFold - 1) / kFold : 0;
        p.bytes = p.o_folds + align_up(static_cast<size_t>(r.N) * p.folded * r.C * 8, 256);
        return p;
    }
    if (backward) {
        p.parts = p.shared ? r.N * p.members
                           : std::min<int64_t>(p.blocks, std::max<int64_t>(1, static_cast<int64_t>(device_cu_count()) * (1024 / p.threads) / p.slabs));
        p.bytes = align_up(static_cast<size_t>(p.parts) * 2 * r.C * 4, 256);
    }
    p.o_exchange = p.bytes;
    if (p.shared) p.bytes += align_up(static_cast<size_t>(r.N) * p.slabs * p.members * p.Gs * 8, 256);
    return p;
}

// The plans of a request's sizes for addresses that are multiples of 16 bytes, of 4, and
// of less.  A thread keeps those that it made last: a step asks for them again four times
// (a microsecond each: a fifth of the time that a step of 256 x 8 x 24 takes to launch).
struct GroupPlans {
    int64_t N = -1, S, C, G;
    int dtype, cus;
    GroupPlan at[3];
    size_t most;                 // bytes of workspace, whatever the addresses
};

const GroupPlans &plans_of(const GroupRequest &r, bool backward) {
    constexpr int kKept = 8;
    thread_local GroupPlans kept[2][kKept];
    const int cus = device_cu_count();
    GroupPlans &k = kept[backward][static_cast<uint64_t>(r.N + 31 * r.S + 7 * r.C + r.dtype) % kKept];
    if (k.N != r.N || k.S != r.S || k.C != r.C || k.G != r.G || k.dtype != r.dtype || k.cus != cus) {
        k.N = r.N; k.S = r.S; k.C = r.C; k.G = r.G; k.dtype = r.dtype; k.cus = cus;
        k.most = 0;
        for (int i = 0; i < 3; ++i) {
            k.at[i] = plan_group(r, backward, i == 0, i <= 1);
            k.most = std::max(k.most, k.at[i].bytes);
        }
    }
    return k;
}

const GroupPlan &plan_group(const GroupRequest &r, bool backward) {
    uintptr_t any = 0;
    for (const void *q : {r.x, r.g, static_cast<const void *>(r.y)}) any |= reinterpret_cast<uintptr_t>(q);
    return plans_of(r, backward).at[any % 16 == 0 ? 0 : (any % 4 == 0 ? 1 : 2)];
}

// How often a member looks for another's values (a microsecond each, about): more than
// any start of workgroups takes that are not kept waiting by other work.
constexpr int kPolls = 4000;

// S rows of P values in shares of `rows` rows
Shares shares_of(int64_t S, int64_t P, int64_t rows) {
    const int64_t last = (S - 1) / rows;
    const double count = static_cast<double>(rows) * P, count_last = static_cast<double>(S - last * rows) * P;
    return {static_cast<float>(count), static_cast<float>(count_last), static_cast<float>(1 / count),
            static_cast<float>(1 / count_last), static_cast<int>(last)};
}

GroupArgs group_args(const GroupRequest &r, const GroupPlan &p) {
    GroupArgs a{};
    a.x = r.x; a.g = r.g; a.weight = r.weight; a.bias = r.bias; a.y = r.y;
    a.stats = reinterpret_cast<float2 *>(r.stats);
    char *ws = static_cast<char *>(r.workspace);
    if (!p.held) {
        a.sums = reinterpret_cast<float2 *>(ws);
        a.channels = reinterpret_cast<float2 *>(ws + p.o_channels);
        a.means = reinterpret_cast<float2 *>(ws + p.o_means);
        a.folds = reinterpret_cast<float2 *>(ws + p.o_folds);
        a.folded = p.folded;
        const int64_t piece_rows = static_cast<int64_t>(p.slots) * kSplitRows;
        a.share = shares_of(r.S, 1, piece_rows);
        a.fold = shares_of(r.S, 1, piece_rows * kFold);
    }
    if (p.shared) {
        a.exchange = reinterpret_cast<uint64_t *>(ws + p.o_exchange);
        a.members = p.members;
        a.member_rows = p.member_rows;
        a.share = shares_of(r.S, r.C / r.G, p.member_rows);
        const int forced = tuning(PLE_TUNE_GROUP_POLLS);
        a.polls = forced > 0 ? forced - 1 : kPolls;
    }
    a.N = r.N; a.S = r.S; a.blocks = p.blocks;
    a.C = static_cast<int>(r.C); a.G = static_cast<int>(r.G); a.P = static_cast<int>(r.C / r.G);
    a.L = p.L; a.slots = p.slots; a.A = p.L * p.slots; a.U = p.U;
    a.slabs = p.slabs; a.Cs = p.Cs; a.Gs = p.Gs;
    a.team = p.team; a.pieces = p.pieces;
    const int64_t wide = p.whole ? r.C / r.G / p.E : r.C / r.G;
    a.wide_inverse = static_cast<uint32_t>(std::min<int64_t>(UINT32_MAX, ((int64_t{1} << 32) + wide - 1) / wide));
    a.act = r.act; a.param_dtype = r.param_dtype;
    a.param_vectors = p.words == 4 && reinterpret_cast<uintptr_t>(r.weight) % 16 == 0 && reinterpret_cast<uintptr_t>(r.bias) % 16 == 0;
    a.eps = r.eps;
    a.inv = static_cast<float>(1.0 / (static_cast<double>(r.S) * static_cast<double>(r.C / r.G)));
    return a;
}

// f(type, words) as compile-time constants
template <typename F>
hipError_t with_piece(int dtype, int words, F f) {
    const auto by_words = [&](auto t) {
        constexpr int T = decltype(t)::value;
        if (words == 4) return f(t, std::integral_constant<int, 4>{});
        if (T == PLE_DTYPE_F32 || words == 1) return f(t, std::integral_constant<int, 1>{});
        if constexpr (T != PLE_DTYPE_F32) return f(t, std::integral_constant<int, 0>{});
        return hipErrorInvalidValue;
    };
    if (dtype == PLE_DTYPE_F32) return by_words(std::integral_constant<int, PLE_DTYPE_F32>{});
    if (dtype == PLE_DTYPE_F16) return by_words(std::integral_constant<int, PLE_DTYPE_F16>{});
    return by_words(std::integral_constant<int, PLE_DTYPE_BF16>{});
}

// f(type, words, whole, threads, rows, shared)
template <const HeldShape *SHAPES, typename F>
hipError_t with_held(int dtype, const GroupPlan &p, F f) {
    return with_piece(dtype, p.words, [&](auto t, auto w) {
        constexpr int W = decltype(w)::value, E = Piece<decltype(t)::value, W>::kElems;
        const auto by_shape = [&](auto whole) {
            const auto at = [&](auto i, auto shared) {
                constexpr HeldShape s = SHAPES[decltype(i)::value];
                return f(t, w, whole, std::integral_constant<int, s.threads>{}, std::integral_constant<int, rows_of(s, W, decltype(shared)::value)>{}, shared);
            };
            using Last = std::integral_constant<int, kShapes - 1>;
            if (p.shared) return at(Last{}, std::true_type{});
            const auto is = [&](int i) { return p.threads == SHAPES[i].threads && p.rows == rows_of(SHAPES[i], W, false); };
            if (is(0)) return at(std::integral_constant<int, 0>{}, std::false_type{});
            if (is(1)) return at(std::integral_constant<int, 1>{}, std::false_type{});
            if (is(2)) return at(std::integral_constant<int, 2>{}, std::false_type{});
            return at(Last{}, std::false_type{});
        };
        if constexpr (E == 1) return by_shape(std::true_type{});
        else if constexpr (E == 2) return by_shape(std::false_type{});
        else return p.whole ? by_shape(std::true_type{}) : by_shape(std::false_type{});
    });
}

// (a grid stays below 2^32 threads; workgroups walk what is left)
constexpr int64_t kMaxGrid = 1 << 20;

dim3 split_grid(const GroupPlan &p) { return dim3(static_cast<unsigned>(std::min<int64_t>(p.blocks, kMaxGrid))); }

bool bad_workspace(const GroupRequest &r, size_t need) {
    return need > 0 && (!r.workspace || r.workspace_bytes < need || reinterpret_cast<uintptr_t>(r.workspace) % 256 != 0);
}

// (by a kernel: a captured graph holds no clearing of memory)
hipError_t clear_exchange(const GroupRequest &r, const GroupPlan &p, const GroupArgs &a) {
    if (!p.shared) return hipSuccess;
    const int64_t n = r.N * p.slabs * p.members * p.Gs;
    hipLaunchKernelGGL(ple_group_unknown_kernel, dim3(static_cast<unsigned>(std::min<int64_t>((n + kBlock - 1) / kBlock, 1024))),
                       dim3(kBlock), 0, r.stream, a.exchange, n);
    return hipGetLastError();
}

template <bool CENTRED>
hipError_t fold(const GroupRequest &r, const GroupArgs &a) {
    if (a.folded == 0) return hipSuccess;
    const int64_t blocks = (a.N * a.folded * a.C + kBlock - 1) / kBlock;
    hipLaunchKernelGGL(ple_group_fold_kernel<CENTRED>, dim3(static_cast<unsigned>(std::min(blocks, kMaxGrid))), dim3(kBlock), 0,
                       r.stream, a);
    return hipGetLastError();
}

}  // namespace

// (Before the call's addresses are known: the plan follows their alignment.)
size_t group_workspace_bytes(const GroupRequest &r) { return plans_of(r, false).most; }

size_t group_backward_workspace_bytes(const GroupRequest &r) { return plans_of(r, true).most; }

int group_plan_info(const GroupRequest &r, bool backward, ple_group_norm_plan_info_t *info) {
    *info = ple_group_norm_plan_info_t{};
    if (r.N == 0 || r.S == 0) return PLE_OK;
    const GroupPlan &p = plan_group(r, backward);
    info->form = p.shared ? PLE_GROUP_SHARED : p.held ? PLE_GROUP_HELD : PLE_GROUP_SPLIT;
    info->lane_channels = p.E;
    info->slabs = p.slabs;
    info->members = p.members;
    info->workspace_bytes = backward ? group_backward_workspace_bytes(r) : group_workspace_bytes(r);
    info->params_end = r.C;                      // (held and shared: slabs are of one width)
    if (!p.held) {
        const GroupArgs a = group_args(r, p);
        const auto reach = [&](auto e) {
            constexpr int E = decltype(e)::value;
            for (int slab = 0; slab < p.slabs; ++slab)
                for (int t = 0; t < kBlock; ++t)
                    info->params_end = std::max<int64_t>(info->params_end, SplitChannels<E>::first_param(a, Split(a, E, slab, t).c0) + E);
        };
        if (p.E == 8) reach(std::integral_constant<int, 8>{});
        else if (p.E == 4) reach(std::integral_constant<int, 4>{});
        else if (p.E == 2) reach(std::integral_constant<int, 2>{});
        else reach(std::integral_constant<int, 1>{});
    }
    return PLE_OK;
}

int group_run(const GroupRequest &r) {
    if (bad_workspace(r, group_workspace_bytes(r))) return PLE_E_WORKSPACE;
    const GroupPlan &p = plan_group(r, false);
    const GroupArgs a = group_args(r, p);
    if (p.held) {
        const hipError_t rc = clear_exchange(r, p, a);
        if (rc != hipSuccess) return static_cast<int>(rc);
        const int64_t grid = p.shared ? r.N * p.slabs * p.members
                                      : std::min<int64_t>(p.blocks, std::max<int64_t>(1, kMaxGrid / p.slabs)) * p.slabs;
        return static_cast<int>(with_held<kForwardShapes>(r.dtype, p, [&](auto t, auto w, auto whole, auto threads, auto rows, auto shared) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_group_forward_kernel<decltype(t)::value, decltype(w)::value,
                                                                        decltype(whole)::value, decltype(threads)::value,
                                                                        decltype(rows)::value, decltype(shared)::value>),
                               dim3(static_cast<unsigned>(grid)), dim3(decltype(threads)::value), p.lds, r.stream, a);
            return hipGetLastError();
        }));
    }
    return static_cast<int>(with_piece(r.dtype, p.words, [&](auto t, auto w) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_group_sums_kernel<decltype(t)::value, decltype(w)::value>), split_grid(p),
                           dim3(kBlock), p.lds, r.stream, a);
        hipError_t rc = hipGetLastError();
        if (rc == hipSuccess) rc = fold<true>(r, a);
        if (rc != hipSuccess) return rc;
        hipLaunchKernelGGL(ple_group_stats_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(r.N * r.G, kMaxGrid))),
                           dim3(kBlock), 0, r.stream, folded_args(a));
        rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_group_apply_kernel<decltype(t)::value, decltype(w)::value>), split_grid(p),
                           dim3(kBlock), 0, r.stream, a);
        return hipGetLastError();
    }));
}

int group_backward_run(const GroupRequest &r) {
    const bool params = r.d_bias || r.d_weight, rows = r.N > 0 && r.S > 0;
    if (rows && bad_workspace(r, group_backward_workspace_bytes(r))) return PLE_E_WORKSPACE;
    const GroupPlan p = rows ? plan_group(r, true) : GroupPlan{};
    GroupArgs a = rows ? group_args(r, p) : GroupArgs{};
    ParamJoin j{};                   // (without rows of no parts: the gradients are 0)
    j.bias = r.d_bias; j.weight = r.d_weight;
    j.C = static_cast<int>(r.C); j.param_dtype = r.param_dtype;
    hipError_t rc = hipSuccess;
    if (rows && p.held) {
        a.partial = params ? static_cast<float *>(r.workspace) : nullptr;
        rc = clear_exchange(r, p, a);
        if (rc != hipSuccess) return static_cast<int>(rc);
        const int64_t grid = p.shared ? r.N * p.slabs * p.members : p.parts * p.slabs;
        rc = with_held<kBackwardShapes>(r.dtype, p, [&](auto t, auto w, auto whole, auto threads, auto rows, auto shared) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_group_backward_kernel<decltype(t)::value, decltype(w)::value,
                                                                         decltype(whole)::value, decltype(threads)::value,
                                                                         decltype(rows)::value, decltype(shared)::value>),
                               dim3(static_cast<unsigned>(grid)), dim3(decltype(threads)::value), p.lds, r.stream, a);
            return hipGetLastError();
        });
        j.sums = a.partial;
        j.parts = p.parts; j.part_stride = 2 * r.C; j.sum_stride = r.C; j.step = 1;
    } else if (rows) {
        rc = with_piece(r.dtype, p.words, [&](auto t, auto w) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_group_backward_sums_kernel<decltype(t)::value, decltype(w)::value>),
                               split_grid(p), dim3(kBlock), p.lds, r.stream, a);
            hipError_t e = hipGetLastError();
            if (e == hipSuccess) e = fold<false>(r, a);
            if (e != hipSuccess) return e;
            hipLaunchKernelGGL(ple_group_backward_join_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(r.N * r.G, kMaxGrid))),
                               dim3(kBlock), 0, r.stream, folded_args(a));
            e = hipGetLastError();
            if (e != hipSuccess || !r.y) return e;
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_group_backward_apply_kernel<decltype(t)::value, decltype(w)::value>),
                               split_grid(p), dim3(kBlock), 0, r.stream, a);
            return hipGetLastError();
        });
        j.sums = reinterpret_cast<const float *>(a.channels);
        j.parts = r.N; j.part_stride = 2 * r.C; j.sum_stride = 1; j.step = 2;
    }
    if (rc != hipSuccess || !params) return static_cast<int>(rc);
    hipLaunchKernelGGL(ple_group_param_kernel, dim3(static_cast<unsigned>((j.C + kParamChannels - 1) / kParamChannels), 2),
                       dim3(kParamThreads), 0, r.stream, j);
    return static_cast<int>(hipGetLastError());
}

}  // namespace ple

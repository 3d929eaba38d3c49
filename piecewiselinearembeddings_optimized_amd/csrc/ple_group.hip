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
// Split form, for samples larger than that: sums of pieces of rows (per channel,
// the squares about the piece's own mean), a join per group, and a second read
// that applies it.

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
    __device__ __forceinline__ void load(const void *p, int64_t i) {
        const char *q = static_cast<const char *>(p) + i * elem_bytes(T);
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
};

template <int T, int W>
__device__ __forceinline__ void store_piece(void *p, int64_t i, const float *v) {
    store_out<T, Piece<T, W>::kElems, false>(p, i, v);
}

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
    int pieces, parts;
    int act, param_dtype;
    float eps, inv;              // inv: 1 / (S P)
};

// ---------------------------------------------------------------------------
// activations
// ---------------------------------------------------------------------------

// Standard normal distribution and density at z.
__device__ __forceinline__ void normal_cdf(float z, float &cdf, float &pdf) {
    cdf = 0.5f * (1.0f + erff(z * 0.70710678118654752f));
    pdf = 0.39894228040143268f * __expf(-0.5f * z * z);
}

__device__ __forceinline__ float logistic(float z) { return 1.0f / (1.0f + __expf(-z)); }

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
            z[e] = s + z[e] * s * (1.0f - s);
        }
    } else if (act == PLE_ACT_GELU) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float cdf, pdf;
            normal_cdf(z[e], cdf, pdf);
            z[e] = cdf + z[e] * pdf;
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
    int unit, slot, lane;
    bool on;
    __device__ __forceinline__ explicit Place(const GroupArgs &a) {
        unit = threadIdx.x / a.A;
        const int r = threadIdx.x - unit * a.A;
        slot = r / a.L;
        lane = r - slot * a.L;
        on = unit < a.U;
    }
};

// What a lane's channels are: their parameters, and each one's group (WHOLE: one
// group for the whole piece).
template <int E, bool WHOLE>
struct Channels {
    static constexpr int kGroups = WHOLE ? 1 : E;
    float w[E], b[E];
    int group[kGroups];
    __device__ __forceinline__ Channels(const GroupArgs &a, int c0, int local) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool on = c0 + e < a.C;
            w[e] = on && a.weight ? load_any(a.weight, c0 + e, a.param_dtype) : 1.0f;
            b[e] = on && a.bias ? load_any(a.bias, c0 + e, a.param_dtype) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < kGroups; ++e) group[e] = (local + e) / a.P;
    }
    __device__ __forceinline__ int of(int e) const { return group[WHOLE ? 0 : e]; }
};

// Joins the workgroup's per-lane values (WHOLE: one a lane, else one a channel)
// over each group: the values of a group lie next to each other in LDS, a team of
// lanes adds them, and `done(group, sum)` runs on the team's first lane.  K values
// are joined at once.
template <int K, int E, bool WHOLE, int THREADS, typename F>
__device__ __forceinline__ void join_groups(const GroupArgs &a, const Place &p, float *lds, const float (&v)[K][WHOLE ? 1 : E],
                                            F done) {
    constexpr int kEach = WHOLE ? 1 : E;
    const int per = (WHOLE ? a.P / E : a.P) * a.slots;           // values of a group
    const int all = a.U * a.Gs;
    const int plane = a.U * a.A * kEach;
    if (p.on)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                lds[k * plane + p.unit * a.A * kEach + (p.lane * kEach + e) * a.slots + p.slot] = v[k][e];
    __syncthreads();
    const int lane = threadIdx.x & (a.team - 1), teams = THREADS / a.team;
    for (int q0 = 0; q0 < all; q0 += teams) {
        const int q = q0 + threadIdx.x / a.team;
        float s[K] = {};
        if (q < all)
            for (int i = lane; i < per; i += a.team)
#pragma unroll
                for (int k = 0; k < K; ++k) s[k] += lds[k * plane + q * per + i];
#pragma unroll
        for (int k = 0; k < K; ++k) s[k] = group_sum_rt(s[k], a.team);
        if (q < all && lane == 0) done(q, s);
    }
    __syncthreads();
}

// LDS floats of the held form's workgroup.
__host__ __device__ inline int held_floats(int threads, int each, int values, int groups) {
    return threads * each * values + 2 * groups;
}

template <int T, int W, bool WHOLE, int THREADS, int R>
__global__ __launch_bounds__(THREADS) void ple_group_forward_kernel(GroupArgs a) {
    constexpr int E = Piece<T, W>::kElems, kEach = WHOLE ? 1 : E;
    extern __shared__ float s_lds[];
    float *const s_mean = s_lds + a.U * a.A * kEach, *const s_rho = s_mean + a.U * a.Gs;
    const Place p(a);
    const int slab = blockIdx.x % a.slabs;
    const int c0 = slab * a.Cs + p.lane * E;
    const Channels<E, WHOLE> ch(a, c0, p.lane * E);
    for (int64_t blk = blockIdx.x / a.slabs; blk < a.blocks; blk += gridDim.x / a.slabs) {
        const int64_t n = blk * a.U + p.unit;
        const bool on = p.on && n < a.N;
        const int64_t first = (n * a.S + p.slot) * a.C + c0, step = static_cast<int64_t>(a.slots) * a.C;
        Piece<T, W> x[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            x[k].clear();
            if (on && p.slot + k * a.slots < a.S) x[k].load(a.x, first + k * step);
        }
        float v[1][kEach] = {};
#pragma unroll
        for (int k = 0; k < R; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) v[0][WHOLE ? 0 : e] += x[k][e];
        join_groups<1, E, WHOLE, THREADS>(a, p, s_lds, v, [&](int q, const float (&s)[1]) { s_mean[q] = s[0] * a.inv; });
        float mean[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            mean[e] = p.on ? s_mean[p.unit * a.Gs + ch.group[e]] : 0.0f;
            v[0][e] = 0.0f;
        }
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (p.slot + k * a.slots < a.S)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float d = x[k][e] - mean[WHOLE ? 0 : e];
                    v[0][WHOLE ? 0 : e] += d * d;
                }
        join_groups<1, E, WHOLE, THREADS>(a, p, s_lds, v, [&](int q, const float (&s)[1]) {
            const float rho = rsqrtf(s[0] * a.inv + a.eps);
            s_rho[q] = rho;
            const int u = q / a.Gs;
            const int64_t sample = blk * a.U + u;
            if (sample < a.N) a.stats[sample * a.G + slab * a.Gs + (q - u * a.Gs)] = make_float2(s_mean[q], rho);
        });
        float scale[E];
#pragma unroll
        for (int e = 0; e < E; ++e) scale[e] = (p.on ? s_rho[p.unit * a.Gs + ch.of(e)] : 0.0f) * ch.w[e];
#pragma unroll
        for (int k = 0; k < R; ++k)
            if (on && p.slot + k * a.slots < a.S) {
                float z[E];
#pragma unroll
                for (int e = 0; e < E; ++e) z[e] = (x[k][e] - mean[WHOLE ? 0 : e]) * scale[e] + ch.b[e];
                activate(z, a.act);
                store_piece<T, W>(a.y, first + k * step, z);
            }
    }
}

// The parameters' gradient sums of a workgroup's lanes, by channel: a partial.
template <int E, int THREADS>
__device__ __forceinline__ void leave_sums(const GroupArgs &a, const Place &p, float *lds, const float (&v)[2][E], int slab,
                                           int64_t part) {
    const int rows = a.U * a.slots;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        __syncthreads();
        if (p.on)
#pragma unroll
            for (int e = 0; e < E; ++e) lds[(p.lane * E + e) * rows + p.unit * a.slots + p.slot] = v[k][e];
        __syncthreads();
        for (int c = threadIdx.x; c < a.Cs; c += THREADS) {
            float s = 0.0f;
            for (int i = 0; i < rows; ++i) s += lds[c * rows + i];
            a.partial[(part * 2 + k) * a.C + slab * a.Cs + c] = s;
        }
    }
}

template <int T, int W, bool WHOLE, int THREADS, int R>
__global__ __launch_bounds__(THREADS) void ple_group_backward_kernel(GroupArgs a) {
    constexpr int E = Piece<T, W>::kElems, kEach = WHOLE ? 1 : E;
    extern __shared__ float s_lds[];
    float *const s_m1 = s_lds + 2 * a.U * a.A * kEach, *const s_m2 = s_m1 + a.U * a.Gs;
    const Place p(a);
    const int slab = blockIdx.x % a.slabs;
    const int c0 = slab * a.Cs + p.lane * E;
    const Channels<E, WHOLE> ch(a, c0, p.lane * E);
    float all[2][E] = {};
    for (int64_t blk = blockIdx.x / a.slabs; blk < a.blocks; blk += gridDim.x / a.slabs) {
        const int64_t n = blk * a.U + p.unit;
        const bool on = p.on && n < a.N;
        const int64_t first = (n * a.S + p.slot) * a.C + c0, step = static_cast<int64_t>(a.slots) * a.C;
        Piece<T, W> x[R], g[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            x[k].clear();
            g[k].clear();
            if (on && p.slot + k * a.slots < a.S) {
                x[k].load(a.x, first + k * step);
                g[k].load(a.g, first + k * step);
            }
        }
        float2 st[kEach];
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            st[e] = on ? a.stats[n * a.G + slab * a.Gs + ch.group[e]] : make_float2(0.0f, 0.0f);
        float sum[2][E] = {};
        float dz[R][E];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            float xh[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                xh[e] = (x[k][e] - st[WHOLE ? 0 : e].x) * st[WHOLE ? 0 : e].y;
                dz[k][e] = xh[e] * ch.w[e] + ch.b[e];
            }
            slopes(dz[k], a.act);
            const bool row = on && p.slot + k * a.slots < a.S;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                dz[k][e] = row ? dz[k][e] * g[k][e] : 0.0f;
                sum[0][e] += dz[k][e];
                sum[1][e] += row ? dz[k][e] * xh[e] : 0.0f;
            }
        }
        float v[2][kEach] = {};
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                all[j][e] += sum[j][e];
                v[j][WHOLE ? 0 : e] += sum[j][e] * ch.w[e];
            }
        if (a.y) {
            join_groups<2, E, WHOLE, THREADS>(a, p, s_lds, v, [&](int q, const float (&s)[2]) {
                s_m1[q] = s[0] * a.inv;
                s_m2[q] = s[1] * a.inv;
            });
            float m1[kEach], m2[kEach];
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                m1[e] = p.on ? s_m1[p.unit * a.Gs + ch.group[e]] : 0.0f;
                m2[e] = p.on ? s_m2[p.unit * a.Gs + ch.group[e]] : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < R; ++k)
                if (on && p.slot + k * a.slots < a.S) {
                    float d[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float2 s = st[WHOLE ? 0 : e];
                        const float xh = (x[k][e] - s.x) * s.y;
                        d[e] = s.y * (dz[k][e] * ch.w[e] - m1[WHOLE ? 0 : e] - xh * m2[WHOLE ? 0 : e]);
                    }
                    store_piece<T, W>(a.y, first + k * step, d);
                }
        }
    }
    if (a.partial) leave_sums<E, THREADS>(a, p, s_lds, all, slab, blockIdx.x / a.slabs);
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
    __device__ __forceinline__ Split(const GroupArgs &a, int E, int64_t blk) {
        slot = threadIdx.x / a.L;
        lane = threadIdx.x - slot * a.L;
        const int64_t u = blk / a.slabs;
        slab = static_cast<int>(blk - u * a.slabs);
        n = u / a.pieces;
        piece = static_cast<int>(u - n * a.pieces);
        row = static_cast<int64_t>(piece) * a.slots * kSplitRows + slot;
        c0 = slab * a.Cs + lane * E;
        on = slot < a.slots && c0 < a.C;
    }
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
        const int64_t rows = min(static_cast<int64_t>(a.slots) * kSplitRows, a.S - static_cast<int64_t>(p.piece) * a.slots * kSplitRows);
        const float inv = 1.0f / static_cast<float>(rows);
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
        const int64_t piece_rows = static_cast<int64_t>(a.slots) * kSplitRows;
        for (int64_t i = threadIdx.x; i < all; i += kBlock) {
            const int64_t piece = i / a.P;
            const float2 s = sums[piece * a.C + i % a.P];
            const float rows = static_cast<float>(min(piece_rows, a.S - piece * piece_rows));
            const float d = s.x / rows - mean;
            t += s.y + rows * d * d;
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
        const Channels<E, false> ch(a, p.c0, p.c0);
        float mean[E], scale[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float2 s = a.stats[p.n * a.G + min(ch.of(e), a.G - 1)];
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
                for (int e = 0; e < E; ++e) z[e] = (x[k][e] - mean[e]) * scale[e] + ch.b[e];
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
        const Channels<E, false> ch(a, p.c0, p.c0);
        float v[E] = {}, u[E] = {};
        if (p.on) {
            float2 st[E];
#pragma unroll
            for (int e = 0; e < E; ++e) st[e] = a.stats[p.n * a.G + min(ch.of(e), a.G - 1)];
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
                        xh[e] = (x[k][e] - st[e].x) * st[e].y;
                        dz[e] = xh[e] * ch.w[e] + ch.b[e];
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
        const Channels<E, false> ch(a, p.c0, p.c0);
        float2 st[E], m[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            st[e] = a.stats[p.n * a.G + min(ch.of(e), a.G - 1)];
            m[e] = a.means[p.n * a.G + min(ch.of(e), a.G - 1)];
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
                    xh[e] = (x[k][e] - st[e].x) * st[e].y;
                    dz[e] = xh[e] * ch.w[e] + ch.b[e];
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

constexpr int kJoinWaves = 16;

struct ParamJoin {
    const float *sums;           // sum k (0: dz, 1: dz xh) of channel c of a part: sums[part * part_stride + k * sum_stride + c * step]
    void *bias, *weight;
    int64_t parts, part_stride, sum_stride;
    int step, C, param_dtype;
};

// 64 channels a workgroup, its waves a part each in turn; blockIdx.y: which sum
__global__ __launch_bounds__(kJoinWaves * kWave) void ple_group_param_kernel(ParamJoin a) {
    __shared__ float s_sum[kJoinWaves * kWave];
    const int wave = threadIdx.x / kWave, c = blockIdx.x * kWave + threadIdx.x % kWave, k = blockIdx.y;
    float v = 0.0f;
    if (c < a.C) {
#pragma unroll 8
        for (int64_t p = wave; p < a.parts; p += kJoinWaves)
            v += a.sums[p * a.part_stride + k * a.sum_stride + static_cast<int64_t>(c) * a.step];
    }
    s_sum[threadIdx.x] = v;
    __syncthreads();
    void *const out = k == 0 ? a.bias : a.weight;
    if (wave == 0 && c < a.C && out) {
        for (int w = 1; w < kJoinWaves; ++w) v += s_sum[w * kWave + threadIdx.x];
        store_any(out, c, v, a.param_dtype);
    }
}

// ---------------------------------------------------------------------------
// plans and launches
// ---------------------------------------------------------------------------

struct GroupPlan {
    int words;                   // a lane's piece: 4, 1 or 0 dwords
    int E;
    bool whole, held;
    int threads, rows;           // held: threads and rows a lane (both compile-time)
    int L, slots, U, slabs, Cs, Gs, team, pieces;
    int64_t blocks, parts;
    size_t lds, o_sums, o_channels, o_means, bytes;
};

// The widest piece that divides a row's slab and its address.
int piece_words(int dtype, int64_t channels, bool aligned16, bool aligned4) {
    const int64_t bytes = channels * elem_bytes(dtype);
    if (aligned16 && bytes % 16 == 0) return 4;
    if (aligned4 && bytes % 4 == 0) return 1;
    return 0;
}

int piece_elems(int dtype, int words) { return words == 0 ? 1 : (dtype == PLE_DTYPE_F32 ? words : 2 * words); }

// The workgroups and rows a lane of the held form.
struct HeldShape {
    int threads, rows;
};
constexpr HeldShape kForwardShapes[] = {{64, 4}, {64, 16}, {256, 16}, {1024, 16}};
constexpr HeldShape kBackwardShapes[] = {{64, 4}, {256, 4}, {256, 8}, {512, 8}};

// The smallest workgroup that holds S rows of Cs channels, or false.
bool held_shape(const HeldShape *shapes, int count, int64_t S, int L, HeldShape &out, int &slots) {
    for (int i = 0; i < count; ++i) {
        if (L > shapes[i].threads) continue;
        const int64_t at_once = std::min<int64_t>(S, shapes[i].threads / L);
        if (at_once * shapes[i].rows < S) continue;
        out = shapes[i];
        slots = static_cast<int>((S + shapes[i].rows - 1) / shapes[i].rows);      // as few as hold them ...
        slots = static_cast<int>(std::max<int64_t>(slots, at_once));              // ... but as many as there are lanes for
        return true;
    }
    return false;
}

GroupPlan plan_group(const GroupRequest &r, bool backward, bool aligned16, bool aligned4) {
    GroupPlan p{};
    const int64_t P = r.C / r.G;
    const HeldShape *shapes = backward ? kBackwardShapes : kForwardShapes;
    // held: as many groups a workgroup as fit; a slab's part of a row is a cache line or more
    for (int64_t gs = r.G; gs >= 1 && !p.held; --gs) {
        if (r.G % gs != 0) continue;
        const int64_t Cs = gs * P;
        if (gs < r.G && Cs * elem_bytes(r.dtype) < 128) break;
        const int words = piece_words(r.dtype, gs < r.G ? Cs : r.C, aligned16, aligned4);
        if (gs < r.G && words != 4) continue;
        const int E = piece_elems(r.dtype, words);
        const int64_t L = Cs / E;
        HeldShape shape{};
        int slots = 0;
        if (L > 1024 || !held_shape(shapes, 4, r.S, static_cast<int>(L), shape, slots)) continue;
        p.held = true;
        p.words = words; p.E = E; p.whole = E != 2 && P % E == 0;      // (with_held's kernels)
        p.threads = shape.threads; p.rows = shape.rows;
        p.L = static_cast<int>(L); p.slots = slots;
        p.slabs = static_cast<int>(r.G / gs); p.Cs = static_cast<int>(Cs); p.Gs = static_cast<int>(gs);
        const int A = p.L * p.slots;
        p.U = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(p.threads / A, r.N)));
        p.blocks = (r.N + p.U - 1) / p.U;
        const int each = p.whole ? 1 : E, values = static_cast<int>((p.whole ? P / E : P) * p.slots), groups = p.U * p.Gs;
        p.team = 1;
        while (p.team < kWave && 2 * p.team * groups <= p.threads && 2 * p.team <= values) p.team *= 2;
        size_t floats = held_floats(p.threads, each, backward ? 2 : 1, groups);
        if (backward) floats = std::max<size_t>(floats, static_cast<size_t>(p.U) * A * E);
        p.lds = floats * 4;
        if (p.lds > kLdsMax) p.held = false;
    }
    if (!p.held) {
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
        p.bytes = p.o_means + (backward ? align_up(static_cast<size_t>(r.N) * r.G * 8, 256) : 0);
        return p;
    }
    if (backward) {
        p.parts = std::min<int64_t>(p.blocks, std::max<int64_t>(1, static_cast<int64_t>(device_cu_count()) * (1024 / p.threads) / p.slabs));
        p.bytes = align_up(static_cast<size_t>(p.parts) * 2 * r.C * 4, 256);
    }
    return p;
}

GroupPlan plan_group(const GroupRequest &r, bool backward) {
    bool a16 = true, a4 = true;
    for (const void *q : {r.x, r.g, static_cast<const void *>(r.y)}) {
        a16 = a16 && reinterpret_cast<uintptr_t>(q) % 16 == 0;
        a4 = a4 && reinterpret_cast<uintptr_t>(q) % 4 == 0;
    }
    return plan_group(r, backward, a16, a4);
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
    }
    a.N = r.N; a.S = r.S; a.blocks = p.blocks;
    a.C = static_cast<int>(r.C); a.G = static_cast<int>(r.G); a.P = static_cast<int>(r.C / r.G);
    a.L = p.L; a.slots = p.slots; a.A = p.L * p.slots; a.U = p.U;
    a.slabs = p.slabs; a.Cs = p.Cs; a.Gs = p.Gs;
    a.team = p.team; a.pieces = p.pieces;
    a.act = r.act; a.param_dtype = r.param_dtype;
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

// f(type, words, whole, threads, rows)
template <const HeldShape *SHAPES, typename F>
hipError_t with_held(int dtype, const GroupPlan &p, F f) {
    return with_piece(dtype, p.words, [&](auto t, auto w) {
        constexpr int E = Piece<decltype(t)::value, decltype(w)::value>::kElems;
        const auto by_shape = [&](auto whole) {
            const auto at = [&](auto i) {
                constexpr HeldShape s = SHAPES[decltype(i)::value];
                return f(t, w, whole, std::integral_constant<int, s.threads>{}, std::integral_constant<int, s.rows>{});
            };
            if (p.threads == SHAPES[0].threads && p.rows == SHAPES[0].rows) return at(std::integral_constant<int, 0>{});
            if (p.threads == SHAPES[1].threads && p.rows == SHAPES[1].rows) return at(std::integral_constant<int, 1>{});
            if (p.threads == SHAPES[2].threads && p.rows == SHAPES[2].rows) return at(std::integral_constant<int, 2>{});
            return at(std::integral_constant<int, 3>{});
        };
        if constexpr (E == 1) return by_shape(std::true_type{});
        else if constexpr (E == 2) return by_shape(std::false_type{});
        else return p.whole ? by_shape(std::true_type{}) : by_shape(std::false_type{});
    });
}

// (a grid stays below 2^32 threads; workgroups walk what is left)
constexpr int64_t kMaxGrid = 1 << 20;

dim3 split_grid(const GroupPlan &p) { return dim3(static_cast<unsigned>(std::min<int64_t>(p.blocks, kMaxGrid))); }

bool bad_workspace(const GroupRequest &r, const GroupPlan &p) {
    return p.bytes > 0 && (!r.workspace || r.workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(r.workspace) % 256 != 0);
}

template <typename F>
size_t most_bytes(const GroupRequest &r, F plan) {
    return std::max({plan(true, true), plan(false, true), plan(false, false)});
}

}  // namespace

// (Before the call's addresses are known: the plan follows their alignment.)
size_t group_workspace_bytes(const GroupRequest &r) {
    return most_bytes(r, [&](bool a16, bool a4) { return plan_group(r, false, a16, a4).bytes; });
}

size_t group_backward_workspace_bytes(const GroupRequest &r) {
    return most_bytes(r, [&](bool a16, bool a4) { return plan_group(r, true, a16, a4).bytes; });
}

int group_run(const GroupRequest &r) {
    const GroupPlan p = plan_group(r, false);
    if (bad_workspace(r, p)) return PLE_E_WORKSPACE;
    const GroupArgs a = group_args(r, p);
    if (p.held) {
        const int64_t grid = std::min<int64_t>(p.blocks, std::max<int64_t>(1, kMaxGrid / p.slabs)) * p.slabs;
        return static_cast<int>(with_held<kForwardShapes>(r.dtype, p, [&](auto t, auto w, auto whole, auto threads, auto rows) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_group_forward_kernel<decltype(t)::value, decltype(w)::value,
                                                                        decltype(whole)::value, decltype(threads)::value,
                                                                        decltype(rows)::value>),
                               dim3(static_cast<unsigned>(grid)), dim3(decltype(threads)::value), p.lds, r.stream, a);
            return hipGetLastError();
        }));
    }
    return static_cast<int>(with_piece(r.dtype, p.words, [&](auto t, auto w) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_group_sums_kernel<decltype(t)::value, decltype(w)::value>), split_grid(p),
                           dim3(kBlock), p.lds, r.stream, a);
        hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
        hipLaunchKernelGGL(ple_group_stats_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(r.N * r.G, kMaxGrid))), dim3(kBlock), 0, r.stream, a);
        rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_group_apply_kernel<decltype(t)::value, decltype(w)::value>), split_grid(p),
                           dim3(kBlock), 0, r.stream, a);
        return hipGetLastError();
    }));
}

int group_backward_run(const GroupRequest &r) {
    const bool params = r.d_bias || r.d_weight, rows = r.N > 0 && r.S > 0;
    const GroupPlan p = rows ? plan_group(r, true) : GroupPlan{};
    if (bad_workspace(r, p)) return PLE_E_WORKSPACE;
    GroupArgs a = rows ? group_args(r, p) : GroupArgs{};
    ParamJoin j{};                   // (without rows of no parts: the gradients are 0)
    j.bias = r.d_bias; j.weight = r.d_weight;
    j.C = static_cast<int>(r.C); j.param_dtype = r.param_dtype;
    hipError_t rc = hipSuccess;
    if (rows && p.held) {
        a.partial = params ? static_cast<float *>(r.workspace) : nullptr;
        rc = with_held<kBackwardShapes>(r.dtype, p, [&](auto t, auto w, auto whole, auto threads, auto rows) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_group_backward_kernel<decltype(t)::value, decltype(w)::value,
                                                                         decltype(whole)::value, decltype(threads)::value,
                                                                         decltype(rows)::value>),
                               dim3(static_cast<unsigned>(p.parts * p.slabs)), dim3(decltype(threads)::value), p.lds, r.stream, a);
            return hipGetLastError();
        });
        j.sums = a.partial;
        j.parts = p.parts; j.part_stride = 2 * r.C; j.sum_stride = r.C; j.step = 1;
    } else if (rows) {
        rc = with_piece(r.dtype, p.words, [&](auto t, auto w) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_group_backward_sums_kernel<decltype(t)::value, decltype(w)::value>),
                               split_grid(p), dim3(kBlock), p.lds, r.stream, a);
            hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            hipLaunchKernelGGL(ple_group_backward_join_kernel, dim3(static_cast<unsigned>(std::min<int64_t>(r.N * r.G, kMaxGrid))), dim3(kBlock), 0, r.stream, a);
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
    hipLaunchKernelGGL(ple_group_param_kernel, dim3(static_cast<unsigned>((j.C + kWave - 1) / kWave), 2), dim3(kJoinWaves * kWave), 0,
                       r.stream, j);
    return static_cast<int>(hipGetLastError());
}

}  // namespace ple

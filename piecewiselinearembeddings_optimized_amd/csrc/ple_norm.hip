// Norms after and before a block, fused with its gate and residual scale
// (gfx950).  For every row (stream r, branch y, both [N, D]):
//
//     p = post(y)                      post, pre: none, rms or layer norm
//     s = round_R(alpha r + h(gate) p) R: the stream's type, h: identity,
//     n = round_Y(pre(s))                 sigmoid or tanh
//
// The norm before the next block and the whole backward read s as it is
// stored, so that they agree with each other.  Backward, with xh the
// standardised row, rho its factor and m() a row's mean:
//
//     ds = dS + rho (dn w - [layer] m(dn w) - xh m(dn w xh))
//     dr = alpha ds,  dp = ds h(gate),  dgate = h'(gate) sum ds p
//     dy = the first line's right term for dp and the norm after the block
//     dw = sum_rows dn xh,  db = sum_rows dn
//
// Bound by memory: forward 2 reads and 2 writes of a row, backward 4 and 2.
// A row is held in registers by a team of lanes, 8 elements each (a part of a
// wave, a wave, or a workgroup of up to 16 waves), so it is read once.  In the
// backward a team walks its rows with the parameters' gradient sums in
// registers; a workgroup adds its teams' sums and leaves them as partials in
// 32 bits, which a second kernel adds in a fixed order.
//
// Measured (one MI355X, kernel trace; forward, backward and joins; the copy's rate
// is 5.2 TB/s): 16384 x 4096 bf16 107 + 164 + 6 us (5.0 and 4.9 TB/s), 51200 x 192
// fp32 34 + 41 + 5 us (4.6 and 5.7: tensors of 39 MB, several of which the
// memory-side cache can hold), 32800 x 1152 fp32 stream with a bf16 branch and a
// gate a sample 92 + 172 + 2 x 5 us (4.9 and 4.0: 144 of 192 lanes, and the biases'
// sums leave three waves a SIMD).  Loads of the next row while this one is used:
// 445 -> 332 us for the first, a second workgroup a CU 332 -> 281.
// Not as near: rows that are not 16-byte vectors load an element at a time (16384 x
// 4100 bf16 548 + 908 us, by vectors at 4096 107 + 164; 65536 x 1001 447 + 645).

#include <algorithm>

#include "ple_internal.h"
#include "ple_rows.h"

namespace ple {
namespace {

constexpr int kElems = 8;              // elements of a row a lane holds
constexpr int kMaxD = 16 * kWave * kElems;

struct NormArgs {
    const void *residual, *branch;     // backward: residual is the stored stream
    const void *post_w, *post_b, *gate, *pre_w, *pre_b;
    void *stream_out, *normed;
    float4 *stats;                     // [N]: mean and factor after the block, before the next
    const void *g_stream, *g_normed;
    void *d_residual, *d_branch, *d_gate;
    float *partial;                    // [workgroups, sums, D]
    float *gate_partial;               // [groups, pieces, D]
    int64_t N, rows_per_gate;
    int64_t block_rows;                // forward: rows of a workgroup
    int64_t piece_rows, pieces;        // backward: rows of a piece, pieces of a gate's rows
    int D, param_dtype;
    int post, pre, act, gates;         // gates: 0 none, 1 one for all rows, 2 one each for groups of rows, 3 one a row
    int slot_pw, slot_pb, slot_g, slot_nw, slot_nb, slots;   // sums' places in a partial (-1: not wanted)
    float alpha, eps;
};

// A lane's 8 elements of a row: adjacent where rows are 16-byte vectors (VEC),
// else one of every `lanes` elements.
template <bool VEC>
struct Cols {
    int first, step, D;
    __device__ __forceinline__ Cols(int lane, int lanes, int d)
        : first(VEC ? lane * kElems : lane), step(VEC ? 1 : lanes), D(d) {}
    __device__ __forceinline__ bool on(int e) const { return VEC ? first < D : first + e * step < D; }
    __device__ __forceinline__ int at(int e) const { return first + e * step; }

    template <int T>
    __device__ __forceinline__ void load(const void *p, int64_t row, float (&v)[kElems]) const {
        if constexpr (VEC) {
            if (on(0)) load_vec<T, kElems>(p, row * D + first, v);
            else
#pragma unroll
                for (int e = 0; e < kElems; ++e) v[e] = 0.0f;
        } else {
#pragma unroll
            for (int e = 0; e < kElems; ++e) v[e] = on(e) ? load_grad<T>(p, row * D + at(e)) : 0.0f;
        }
    }
    template <int T>
    __device__ __forceinline__ void store(void *p, int64_t row, const float (&v)[kElems]) const {
        if constexpr (VEC) {
            if (on(0)) store_vec<T, kElems>(p, row * D + first, v);
        } else {
#pragma unroll
            for (int e = 0; e < kElems; ++e)
                if (on(e)) store_vec<T, 1>(p, row * D + at(e), &v[e]);
        }
    }
    // a row as loaded, widened at use (grad_elem), so that the next row's can be
    // in flight while this one's is used
    template <int T>
    __device__ __forceinline__ void load_raw(const void *p, int64_t row, uint32_t (&w)[grad_words<T, kElems>()]) const {
        constexpr int W = grad_words<T, kElems>();
        if constexpr (VEC) {
            if (on(0)) {
                const uint4 *q = reinterpret_cast<const uint4 *>(static_cast<const char *>(p) + (row * D + first) * elem_bytes(T));
#pragma unroll
                for (int k = 0; k < W / 4; ++k) {
                    const uint4 v = q[k];
                    w[4 * k] = v.x; w[4 * k + 1] = v.y; w[4 * k + 2] = v.z; w[4 * k + 3] = v.w;
                }
            } else {
#pragma unroll
                for (int k = 0; k < W; ++k) w[k] = 0;
            }
        } else {
#pragma unroll
            for (int k = 0; k < W; ++k) w[k] = 0;
#pragma unroll
            for (int e = 0; e < kElems; ++e) {
                if (!on(e)) continue;
                if constexpr (T == PLE_DTYPE_F32) w[e] = static_cast<const uint32_t *>(p)[row * D + at(e)];
                else w[e / 2] |= static_cast<uint32_t>(static_cast<const uint16_t *>(p)[row * D + at(e)]) << (16 * (e % 2));
            }
        }
    }
    // a parameter row of a type known at run time (`none` where there is none)
    __device__ __forceinline__ void load_param(const void *p, int64_t row, int dtype, float none, float (&v)[kElems]) const {
        if (p && dtype == PLE_DTYPE_F32) load<PLE_DTYPE_F32>(p, row, v);
        else if (p && dtype == PLE_DTYPE_BF16) load<PLE_DTYPE_BF16>(p, row, v);
        else if (p) load<PLE_DTYPE_F16>(p, row, v);
        else
#pragma unroll
            for (int e = 0; e < kElems; ++e) v[e] = none;
    }
    __device__ __forceinline__ void store_param(void *p, int64_t row, int dtype, const float (&v)[kElems]) const {
        if (dtype == PLE_DTYPE_F32) store<PLE_DTYPE_F32>(p, row, v);
        else if (dtype == PLE_DTYPE_BF16) store<PLE_DTYPE_BF16>(p, row, v);
        else store<PLE_DTYPE_F16>(p, row, v);
    }
};

__device__ __forceinline__ float gate_value(float x, int act) {
    if (act == PLE_GATE_SIGMOID) return 1.0f / (1.0f + expf(-x));
    if (act == PLE_GATE_TANH) return tanhf(x);
    return x;
}

// Derivative of gate_value, from its value.
__device__ __forceinline__ float gate_slope(float h, int act) {
    if (act == PLE_GATE_SIGMOID) return h * (1.0f - h);
    if (act == PLE_GATE_TANH) return 1.0f - h * h;
    return 1.0f;
}

// Mean (0 for an rms norm) and factor of a row.
template <int TEAM, bool VEC>
__device__ __forceinline__ void row_stats(Team<TEAM> &team, const Cols<VEC> &c, const float (&v)[kElems], int kind,
                                          float eps, float &mean, float &rho) {
    const float inv = 1.0f / static_cast<float>(c.D);
    mean = 0.0f;
    if (kind == PLE_NORM_LAYER) {
        float t = 0.0f;
#pragma unroll
        for (int e = 0; e < kElems; ++e) t += v[e];      // (elements past the row are 0)
        mean = team.sum(t) * inv;
    }
    float t = 0.0f;
#pragma unroll
    for (int e = 0; e < kElems; ++e) {
        const float d = c.on(e) ? v[e] - mean : 0.0f;
        t += d * d;
    }
    rho = rsqrtf(team.sum(t) * inv + eps);
}

// A workgroup takes a contiguous range of rows, its teams every so many of them.
template <int R, int Y, int TEAM, bool VEC>
__global__ __launch_bounds__(Team<TEAM>::kThreads) void ple_norm_forward_kernel(NormArgs a) {
    __shared__ float s_sum[Team<TEAM>::kLdsFloats];
    Team<TEAM> team(s_sum);
    const Cols<VEC> c(team.lane(), team.lanes(), a.D);
    const int64_t begin = static_cast<int64_t>(blockIdx.x) * a.block_rows + team.index();
    const int64_t end = min(a.N, static_cast<int64_t>(blockIdx.x + 1) * a.block_rows);
    if (begin >= end) return;        // (a whole team)
    uint32_t raw_s[grad_words<R, kElems>()], raw_y[grad_words<Y, kElems>()] = {};
    c.template load_raw<R>(a.residual, begin, raw_s);
    if (a.branch) c.template load_raw<Y>(a.branch, begin, raw_y);
    float pw[kElems], pb[kElems], nw[kElems], nb[kElems], h[kElems];
    c.load_param(a.post_w, 0, a.param_dtype, 1.0f, pw);
    c.load_param(a.post_b, 0, a.param_dtype, 0.0f, pb);
    c.load_param(a.pre_w, 0, a.param_dtype, 1.0f, nw);
    c.load_param(a.pre_b, 0, a.param_dtype, 0.0f, nb);
    c.load_param(nullptr, 0, a.param_dtype, 1.0f, h);
    int64_t gate_end = a.gates ? 0 : a.N;        // rows up to here have the gate row in h
    for (int64_t n = begin; n < end; n += team.per_block()) {
        uint32_t next_s[grad_words<R, kElems>()] = {}, next_y[grad_words<Y, kElems>()] = {};
        if (n + team.per_block() < end) {
            c.template load_raw<R>(a.residual, n + team.per_block(), next_s);
            if (a.branch) c.template load_raw<Y>(a.branch, n + team.per_block(), next_y);
        }
        float4 st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
        float s[kElems], v[kElems];
#pragma unroll
        for (int e = 0; e < kElems; ++e) {
            s[e] = grad_elem<R>(raw_s, e);
            v[e] = grad_elem<Y>(raw_y, e);
        }
        if (a.branch) {
            if (n >= gate_end) {
                const int64_t row = n / a.rows_per_gate;
                gate_end = (row + 1) * a.rows_per_gate;
                c.load_param(a.gate, row, a.param_dtype, 1.0f, h);
#pragma unroll
                for (int e = 0; e < kElems; ++e) h[e] = gate_value(h[e], a.act);
            }
            if (a.post != PLE_NORM_NONE) {
                row_stats(team, c, v, a.post, a.eps, st.x, st.y);
#pragma unroll
                for (int e = 0; e < kElems; ++e) v[e] = (v[e] - st.x) * st.y * pw[e] + pb[e];
            }
#pragma unroll
            for (int e = 0; e < kElems; ++e) s[e] = c.on(e) ? quant<R>(a.alpha * s[e] + h[e] * v[e]) : 0.0f;
            c.template store<R>(a.stream_out, n, s);
        }
        if (a.pre != PLE_NORM_NONE) {
            row_stats(team, c, s, a.pre, a.eps, st.z, st.w);
#pragma unroll
            for (int e = 0; e < kElems; ++e) v[e] = (s[e] - st.z) * st.w * nw[e] + nb[e];
            c.template store<Y>(a.normed, n, v);
        }
        if (team.lane() == 0) a.stats[n] = st;
#pragma unroll
        for (int k = 0; k < grad_words<R, kElems>(); ++k) raw_s[k] = next_s[k];
#pragma unroll
        for (int k = 0; k < grad_words<Y, kElems>(); ++k) raw_y[k] = next_y[k];
    }
}

// d of a norm's input from d of its output (times its weight), in place.
template <int TEAM, bool VEC>
__device__ __forceinline__ void norm_grad(Team<TEAM> &team, const Cols<VEC> &c, float (&g)[kElems],
                                          const float (&xh)[kElems], float rho, int kind) {
    float proj = 0.0f, mean = 0.0f;
#pragma unroll
    for (int e = 0; e < kElems; ++e) {
        proj += g[e] * xh[e];
        mean += g[e];
    }
    team.sum2(proj, mean);
    const float inv = 1.0f / static_cast<float>(c.D);
    proj *= inv;
    mean = kind == PLE_NORM_LAYER ? mean * inv : 0.0f;
#pragma unroll
    for (int e = 0; e < kElems; ++e) g[e] = rho * (g[e] - mean - xh[e] * proj);
}

// A row's inputs of the backward, as loaded.
template <int R, int Y>
struct BackRow {
    uint32_t ds[grad_words<R, kElems>()], x[grad_words<R, kElems>()];
    uint32_t gn[grad_words<Y, kElems>()], y[grad_words<Y, kElems>()];
    float4 st;
    template <bool VEC>
    __device__ __forceinline__ void load(const NormArgs &a, const Cols<VEC> &c, int64_t n) {
        if (a.g_stream) c.template load_raw<R>(a.g_stream, n, ds);
        if (a.g_normed) {
            c.template load_raw<Y>(a.g_normed, n, gn);
            c.template load_raw<R>(a.residual, n, x);
        }
        if (a.branch) c.template load_raw<Y>(a.branch, n, y);
        st = a.stats[n];
    }
};

// A lane's elements of a parameter row over all of its rows: in registers, or
// (LDS) in a place of its own in LDS, two 16-byte reads a use.  The registers of
// wide teams are what keeps a second workgroup off the CU.
template <bool LDS>
struct Held {
    float v[LDS ? 1 : kElems];
    float none = 0.0f;
    float4 *place = nullptr;
    __device__ __forceinline__ void set(const float (&from)[kElems], float *&lds, bool given, float otherwise) {
        if constexpr (LDS) {
            none = otherwise;
            if (!given) return;
            place = reinterpret_cast<float4 *>(lds) + threadIdx.x;
            lds += blockDim.x * kElems;
            place[0] = make_float4(from[0], from[1], from[2], from[3]);
            place[blockDim.x] = make_float4(from[4], from[5], from[6], from[7]);
        } else {
#pragma unroll
            for (int e = 0; e < kElems; ++e) v[e] = from[e];
        }
    }
    __device__ __forceinline__ void get(float (&to)[kElems]) const {
        if constexpr (LDS) {
            if (place) {
                const float4 a = place[0], b = place[blockDim.x];
                to[0] = a.x; to[1] = a.y; to[2] = a.z; to[3] = a.w;
                to[4] = b.x; to[5] = b.y; to[6] = b.z; to[7] = b.w;
            } else {
#pragma unroll
                for (int e = 0; e < kElems; ++e) to[e] = none;
            }
        } else {
#pragma unroll
            for (int e = 0; e < kElems; ++e) to[e] = v[e];
        }
    }
};

// Waves a SIMD the backward of wide rows is compiled for (its registers: 128, 168
// or 256).  Workgroups of up to 768 threads have 168, of more than that 128, which
// with biases are too few (9000 x 5120 layer norms with biases: 547 us with 128,
// 232 with 168).  More than 768 threads can have no more, and spill there (8192 x
// 8192 bf16, backward: 512 us with biases, 162 without).  fp32 rows without biases
// spill up to 53 of 128 registers (16384 x 4096: 486 us of fp32, 3.3 TB/s; 267 of an
// fp32 stream with a bf16 branch, 4.5).
constexpr int backward_waves(bool vec, bool bias) { return !vec ? 2 : bias ? 3 : 4; }

// Teams walk units of rows: a row each, or a piece of the rows of one gate, whose
// sum is finished with the piece.  BIAS: the norms may have biases.  OWN: rows or
// groups of them have gates of their own.
template <int R, int Y, int TEAM, bool VEC, bool BIAS, bool OWN>
__global__ __launch_bounds__(Team<TEAM>::kThreads, TEAM == 512 ? backward_waves(VEC, BIAS) : TEAM == 768 ? 3 : 1) void ple_norm_backward_kernel(NormArgs a) {
    constexpr int kTeams = Team<TEAM>::kBlockWide ? 1 : kBlock / TEAM;
    __shared__ float s_sum[Team<TEAM>::kLdsFloats];
    __shared__ float s_cols[kTeams > 1 ? kBlock * kElems : 1];
    extern __shared__ float s_params[];
    Team<TEAM> team(s_sum);
    const Cols<VEC> c(team.lane(), team.lanes(), a.D);
    const int64_t teams = static_cast<int64_t>(gridDim.x) * team.per_block();
    const int64_t units = a.gates == 2 ? (a.N / a.rows_per_gate) * a.pieces : a.N;
    int64_t u = static_cast<int64_t>(blockIdx.x) * team.per_block() + team.index(), n = 0, stop = 0;
    const auto enter = [&] {         // the rows of unit u
        if (a.gates == 2) {
            const int64_t group = u / a.pieces, piece = u - group * a.pieces;
            n = group * a.rows_per_gate + piece * a.piece_rows;
            stop = min(n + a.piece_rows, (group + 1) * a.rows_per_gate);
        } else {
            n = u;
            stop = u + 1;
        }
    };
    BackRow<R, Y> now{}, next{};
    if (u < units) {
        enter();
        now.load(a, c, n);
    }
    Held<Team<TEAM>::kBlockWide> post_w, post_b, pre_w, gate;
    float h[kElems];                 // OWN: of the unit's rows
    {
        float *lds = s_params, v[kElems];
        c.load_param(a.post_w, 0, a.param_dtype, 1.0f, v);
        post_w.set(v, lds, a.post_w != nullptr, 1.0f);
        if constexpr (BIAS) {
            c.load_param(a.post_b, 0, a.param_dtype, 0.0f, v);
            post_b.set(v, lds, a.post_b != nullptr, 0.0f);
        }
        c.load_param(a.pre_w, 0, a.param_dtype, 1.0f, v);
        pre_w.set(v, lds, a.pre_w != nullptr, 1.0f);
        if constexpr (!OWN) {
            c.load_param(a.gate, 0, a.param_dtype, 1.0f, v);
            if (a.gates)
#pragma unroll
                for (int e = 0; e < kElems; ++e) v[e] = gate_value(v[e], a.act);
            gate.set(v, lds, a.gates != 0, 1.0f);
        }
    }
    float s_pw[kElems] = {}, s_g[kElems] = {}, s_nw[kElems] = {};
    float s_pb[BIAS ? kElems : 1] = {}, s_nb[BIAS ? kElems : 1] = {};
    while (u < units) {
        const int64_t unit = u;
        if constexpr (OWN) {
            c.load_param(a.gate, a.gates == 2 ? unit / a.pieces : unit, a.param_dtype, 1.0f, h);
#pragma unroll
            for (int e = 0; e < kElems; ++e) {
                h[e] = gate_value(h[e], a.act);
                s_g[e] = 0.0f;
            }
        }
        do {
            const int64_t row = n;
            if (++n == stop) {
                u += teams;
                if (u < units) enter();
            }
            if (u < units) next.load(a, c, n);
            const float4 st = now.st;
            float ds[kElems], xh[kElems], g[kElems];
#pragma unroll
            for (int e = 0; e < kElems; ++e) ds[e] = grad_elem<R>(now.ds, e);
            if (a.g_normed) {
                float w[kElems];
                pre_w.get(w);
#pragma unroll
                for (int e = 0; e < kElems; ++e) {
                    g[e] = grad_elem<Y>(now.gn, e);
                    xh[e] = c.on(e) ? (grad_elem<R>(now.x, e) - st.z) * st.w : 0.0f;
                    s_nw[e] += g[e] * xh[e];
                    if constexpr (BIAS) s_nb[e] += g[e];
                    g[e] *= w[e];
                }
                norm_grad(team, c, g, xh, st.w, a.pre);
#pragma unroll
                for (int e = 0; e < kElems; ++e) ds[e] += g[e];
            }
            if (a.d_residual) {
#pragma unroll
                for (int e = 0; e < kElems; ++e) g[e] = a.alpha * ds[e];
                c.template store<R>(a.d_residual, row, g);
            }
            if (a.branch) {
                if constexpr (!OWN) gate.get(h);
#pragma unroll
                for (int e = 0; e < kElems; ++e) xh[e] = grad_elem<Y>(now.y, e);
                if (a.post != PLE_NORM_NONE) {
                    float w[kElems], b[kElems];
                    post_w.get(w);
                    if constexpr (BIAS) post_b.get(b);
#pragma unroll
                    for (int e = 0; e < kElems; ++e) {
                        xh[e] = c.on(e) ? (xh[e] - st.x) * st.y : 0.0f;
                        g[e] = c.on(e) ? ds[e] * h[e] : 0.0f;
                        s_g[e] += ds[e] * (BIAS ? xh[e] * w[e] + b[e] : xh[e] * w[e]);
                        s_pw[e] += g[e] * xh[e];
                        if constexpr (BIAS) s_pb[e] += g[e];
                        g[e] *= w[e];
                    }
                    norm_grad(team, c, g, xh, st.y, a.post);
                } else {
#pragma unroll
                    for (int e = 0; e < kElems; ++e) {
                        g[e] = ds[e] * h[e];
                        s_g[e] += ds[e] * xh[e];
                    }
                }
                if (a.d_branch) c.template store<Y>(a.d_branch, row, g);
            }
            now = next;
        } while (u == unit);
        if constexpr (OWN) {
            if (!a.d_gate) continue;
            float v[kElems];
#pragma unroll
            for (int e = 0; e < kElems; ++e) v[e] = s_g[e] * gate_slope(h[e], a.act);
            if (a.gates == 3 || a.pieces == 1) c.store_param(a.d_gate, unit, a.param_dtype, v);
            else c.template store<PLE_DTYPE_F32>(a.gate_partial, unit, v);
        }
    }
    if constexpr (!OWN) {
        gate.get(h);
#pragma unroll
        for (int e = 0; e < kElems; ++e) s_g[e] *= gate_slope(h[e], a.act);
    }
    const auto leave = [&](float (&v)[kElems], int slot) {
        if (slot < 0) return;
        if constexpr (kTeams > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kElems; ++e) s_cols[e * kBlock + threadIdx.x] = v[e];
            __syncthreads();
            if (team.index() == 0)
                for (int t = 1; t < kTeams; ++t)
#pragma unroll
                    for (int e = 0; e < kElems; ++e) v[e] += s_cols[e * kBlock + t * TEAM + team.lane()];
        }
        if (team.index() == 0)
            c.template store<PLE_DTYPE_F32>(a.partial, static_cast<int64_t>(blockIdx.x) * a.slots + slot, v);
    };
    leave(s_pw, a.slot_pw);
    leave(s_nw, a.slot_nw);
    if constexpr (!OWN) leave(s_g, a.slot_g);
    if constexpr (BIAS) {
        leave(s_pb, a.slot_pb);
        leave(s_nb, a.slot_nb);
    }
}

// out[j, d] = sum over the parts of partial[part, j, d]; 64 columns a workgroup,
// its waves a part each in turn.
constexpr int kJoinWaves = 16;
constexpr int kMaxSums = 5;

struct JoinArgs {
    const float *partial;
    void *out[kMaxSums];         // stacked: out[0] is [sums, D], else one vector a sum
    int64_t part_stride, sum_stride;
    int parts, D, param_dtype, stacked, colblocks;
};

__global__ __launch_bounds__(kJoinWaves * kWave) void ple_norm_join_kernel(JoinArgs a) {
    __shared__ float s_sum[kJoinWaves * kWave];
    const int wave = threadIdx.x / kWave, d = blockIdx.x % a.colblocks * kWave + threadIdx.x % kWave;
    const int64_t j = blockIdx.x / a.colblocks;
    float v = 0.0f;
    if (d < a.D) {
#pragma unroll 8
        for (int p = wave; p < a.parts; p += kJoinWaves) v += a.partial[p * a.part_stride + j * a.sum_stride + d];
    }
    s_sum[threadIdx.x] = v;
    __syncthreads();
    if (wave == 0 && d < a.D) {
        for (int w = 1; w < kJoinWaves; ++w) v += s_sum[w * kWave + threadIdx.x];
        if (a.stacked) store_any(a.out[0], j * a.D + d, v, a.param_dtype);
        else store_any(a.out[j], d, v, a.param_dtype);
    }
}

// ---------------------------------------------------------------------------
// plans and launches
// ---------------------------------------------------------------------------

struct NormPlan {
    int team, threads, per_block, vec;
    int blocks;                          // backward workgroups
    int64_t piece_rows, pieces;
    int slots;
    size_t lds, o_gate, bytes;
};

int gate_mode(const NormRequest &r) {
    if (!r.gate) return 0;
    return r.groups == 1 ? 1 : (r.groups == r.N ? 3 : 2);
}

// aligned: whether every tensor's rows can be read as vectors.
NormPlan plan_norm(const NormRequest &r, bool aligned) {
    NormPlan p{};
    if (r.N == 0) return p;
    const int lanes = static_cast<int>((r.D + kElems - 1) / kElems);
    p.team = lanes <= 8 ? 8 : (lanes <= 16 ? 16 : (lanes <= 32 ? 32 : (lanes <= 64 ? 64 : (lanes <= 512 ? 512 : (lanes <= 768 ? 768 : 1024)))));
    p.threads = p.team > kWave ? (lanes + kWave - 1) / kWave * kWave : kBlock;
    p.per_block = p.team > kWave ? 1 : kBlock / p.team;
    p.vec = aligned && r.D % kElems == 0;
    const int mode = gate_mode(r);
    // as many backward workgroups as run at once (a few more leave most of the GPU
    // idle at the end): by the waves a SIMD has registers for, where workgroups of
    // an odd number of waves fill the four SIMDs as the next multiple of four does
    // (3 waves of 168 registers: 768 workgroups took 175 us where 1024 took 228,
    // 32800 x 1152), and by LDS
    const bool bias = r.post_b || r.pre_b;
    const int simd_waves = p.team == 1024 ? 4 : p.team == 768 ? 3 : p.team < 512 ? (bias ? 2 : 3) : backward_waves(p.vec, bias);
    const int block_waves = p.threads / kWave;
    const int filled = block_waves <= 2 ? block_waves : (block_waves + 3) / 4 * 4;
    p.lds = p.team > kWave ? static_cast<size_t>((r.post_w != nullptr) + (r.post_b != nullptr) + (r.pre_w != nullptr) +
                                                 (mode == 1)) * p.threads * kElems * 4 : 0;
    const int by_lds = p.lds > 0 ? static_cast<int>(kLdsMax / (p.lds + 1024)) : 8;
    const int most = device_cu_count() * std::max(1, std::min(4 * simd_waves / filled, by_lds));
    const int64_t teams = static_cast<int64_t>(most) * p.per_block;
    int64_t units = r.N;
    p.piece_rows = p.pieces = 1;
    if (mode == 2) {
        const int64_t rows = r.N / r.groups;
        // pieces of a gate's rows such that the teams have about one to four each,
        // the most rows a team gets being the fewest
        int64_t best = INT64_MAX;
        for (int64_t k = 1; k <= 4; ++k) {
            const int64_t want = std::min(rows, std::max<int64_t>(1, k * teams / r.groups));
            const int64_t size = (rows + want - 1) / want, pieces = (rows + size - 1) / size;
            const int64_t cost = (r.groups * pieces + teams - 1) / teams * (size + 1);
            if (cost < best) {
                best = cost;
                p.piece_rows = size;
                p.pieces = pieces;
            }
        }
        units = r.groups * p.pieces;
    }
    p.blocks = static_cast<int>(std::min<int64_t>(most, std::max<int64_t>(1, (units + p.per_block - 1) / p.per_block)));
    p.slots = (r.post_w != nullptr) + (r.post_b != nullptr) + (mode == 1) + (r.pre_w != nullptr) + (r.pre_b != nullptr);
    p.o_gate = align_up(static_cast<size_t>(p.blocks) * p.slots * r.D * 4, 256);
    p.bytes = p.o_gate + (mode == 2 && p.pieces > 1 ? align_up(static_cast<size_t>(units) * r.D * 4, 256) : 0);
    return p;
}

NormPlan plan_norm(const NormRequest &r) {
    bool aligned = true;
    for (const void *q : {r.residual, r.branch, r.g_stream, r.g_normed, static_cast<const void *>(r.stream_out),
                          static_cast<const void *>(r.normed), static_cast<const void *>(r.d_residual),
                          static_cast<const void *>(r.d_branch), r.post_w, r.post_b, r.gate, r.pre_w, r.pre_b,
                          static_cast<const void *>(r.d_gate)})
        aligned = aligned && reinterpret_cast<uintptr_t>(q) % 16 == 0;
    return plan_norm(r, aligned);
}

NormArgs norm_args(const NormRequest &r) {
    NormArgs a{};
    a.residual = r.residual; a.branch = r.branch;
    a.post_w = r.post_w; a.post_b = r.post_b; a.gate = r.gate; a.pre_w = r.pre_w; a.pre_b = r.pre_b;
    a.stream_out = r.stream_out; a.normed = r.normed;
    a.stats = reinterpret_cast<float4 *>(r.stats);
    a.g_stream = r.g_stream; a.g_normed = r.g_normed;
    a.d_residual = r.d_residual; a.d_branch = r.d_branch; a.d_gate = r.d_gate;
    a.N = r.N; a.D = static_cast<int>(r.D);
    a.gates = gate_mode(r);
    a.rows_per_gate = a.gates ? r.N / r.groups : r.N;
    a.param_dtype = r.param_dtype;
    a.post = r.post; a.pre = r.pre; a.act = r.act;
    a.alpha = r.alpha; a.eps = r.eps;
    return a;
}

// f(stream type, branch type, team, vectors) as compile-time constants
template <typename F>
hipError_t with_norm(const NormRequest &r, const NormPlan &p, F f) {
    const auto by_vec = [&](auto st, auto br, auto team) {
        return p.vec ? f(st, br, team, std::true_type{}) : f(st, br, team, std::false_type{});
    };
    const auto by_team = [&](auto st, auto br) {
        switch (p.team) {
            case 8: return by_vec(st, br, std::integral_constant<int, 8>{});
            case 16: return by_vec(st, br, std::integral_constant<int, 16>{});
            case 32: return by_vec(st, br, std::integral_constant<int, 32>{});
            case 64: return by_vec(st, br, std::integral_constant<int, 64>{});
            case 512: return by_vec(st, br, std::integral_constant<int, 512>{});
            case 768: return by_vec(st, br, std::integral_constant<int, 768>{});
            default: return by_vec(st, br, std::integral_constant<int, 1024>{});
        }
    };
    using F32 = std::integral_constant<int, PLE_DTYPE_F32>;
    using F16 = std::integral_constant<int, PLE_DTYPE_F16>;
    using BF16 = std::integral_constant<int, PLE_DTYPE_BF16>;
    if (r.stream_dtype == PLE_DTYPE_BF16) return by_team(BF16{}, BF16{});
    if (r.stream_dtype == PLE_DTYPE_F16) return by_team(F16{}, F16{});
    if (r.branch_dtype == PLE_DTYPE_BF16) return by_team(F32{}, BF16{});
    if (r.branch_dtype == PLE_DTYPE_F16) return by_team(F32{}, F16{});
    return by_team(F32{}, F32{});
}

// The gates' joins, of as many gate rows a launch as keep it below 2^32 threads (an
// empty batch can have any number of gate rows).
hipError_t join_gates(const NormRequest &r, JoinArgs j) {
    const int64_t most = (int64_t{1} << 21) / j.colblocks;
    j.stacked = 1;
    for (int64_t g = 0; g < r.groups; g += most) {
        j.out[0] = static_cast<char *>(r.d_gate) + g * r.D * elem_bytes(r.param_dtype);
        hipLaunchKernelGGL(ple_norm_join_kernel, dim3(static_cast<unsigned>(j.colblocks * std::min(most, r.groups - g))),
                           dim3(kJoinWaves * kWave), 0, r.stream, j);
        const hipError_t rc = hipGetLastError();
        if (rc != hipSuccess) return rc;
        j.partial += most * j.sum_stride;
    }
    return hipSuccess;
}

// An empty batch: the parameters' gradients are 0.
int norm_zero_gradients(const NormRequest &r) {
    JoinArgs j{};
    j.D = static_cast<int>(r.D);
    j.param_dtype = r.param_dtype;
    j.colblocks = (j.D + kWave - 1) / kWave;
    int sums = 0;
    for (void *p : {r.d_post_w, r.d_post_b, r.d_pre_w, r.d_pre_b})
        if (p) j.out[sums++] = p;
    if (sums > 0) hipLaunchKernelGGL(ple_norm_join_kernel, dim3(j.colblocks * sums), dim3(kJoinWaves * kWave), 0, r.stream, j);
    const hipError_t rc = hipGetLastError();
    return static_cast<int>(rc == hipSuccess && r.d_gate ? join_gates(r, j) : rc);
}

}  // namespace

int norm_run(const NormRequest &r) {
    if (r.D > kMaxD) return PLE_E_TOO_LARGE;
    const NormPlan p = plan_norm(r);
    NormArgs a = norm_args(r);
    const int64_t most = static_cast<int64_t>(device_cu_count()) * std::max(1, 2048 / p.threads);
    const int64_t steps = (r.N + p.per_block - 1) / p.per_block;
    a.block_rows = (steps + most - 1) / most * p.per_block;
    const dim3 grid(static_cast<unsigned>((r.N + a.block_rows - 1) / a.block_rows));
    return static_cast<int>(with_norm(r, p, [&](auto st, auto br, auto team, auto vec) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_norm_forward_kernel<decltype(st)::value, decltype(br)::value,
                                                                   decltype(team)::value, decltype(vec)::value>),
                           grid, dim3(p.threads), 0, r.stream, a);
        return hipGetLastError();
    }));
}

// (Before the call's addresses are known.  The pieces of gates' rows follow the
// number of workgroups, which is another where vectors are not aligned: either may
// need more.)
size_t norm_backward_workspace_bytes(const NormRequest &r) {
    return r.D > kMaxD ? 0 : std::max(plan_norm(r, true).bytes, plan_norm(r, false).bytes);
}

int norm_backward_run(const NormRequest &r) {
    if (r.D > kMaxD) return PLE_E_TOO_LARGE;
    const NormPlan p = plan_norm(r);
    if (r.N == 0) return norm_zero_gradients(r);
    if (p.bytes > 0 && (!r.workspace || r.workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(r.workspace) % 256 != 0))
        return PLE_E_WORKSPACE;
    NormArgs a = norm_args(r);
    a.piece_rows = p.piece_rows;
    a.pieces = p.pieces;
    a.partial = static_cast<float *>(r.workspace);
    a.gate_partial = reinterpret_cast<float *>(static_cast<char *>(r.workspace) + p.o_gate);
    JoinArgs j{};
    const auto slot = [&](const void *param, void *grad) {
        if (!param || !grad) return -1;
        j.out[a.slots] = grad;
        return a.slots++;
    };
    a.slot_pw = slot(r.post_w, r.d_post_w);
    a.slot_pb = slot(r.post_b, r.d_post_b);
    a.slot_g = slot(a.gates == 1 ? r.gate : nullptr, r.d_gate);
    a.slot_nw = slot(r.pre_w, r.d_pre_w);
    a.slot_nb = slot(r.pre_b, r.d_pre_b);
    const bool bias = r.post_b || r.pre_b, own = a.gates > 1;
    const hipError_t rc = with_norm(r, p, [&](auto st, auto br, auto team, auto vec) {
        const auto launch = [&](auto has_bias, auto has_own) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_norm_backward_kernel<decltype(st)::value, decltype(br)::value,
                                                                        decltype(team)::value, decltype(vec)::value,
                                                                        decltype(has_bias)::value, decltype(has_own)::value>),
                               dim3(p.blocks), dim3(p.threads), p.lds, r.stream, a);
            return hipGetLastError();
        };
        if (bias) return own ? launch(std::true_type{}, std::true_type{}) : launch(std::true_type{}, std::false_type{});
        return own ? launch(std::false_type{}, std::true_type{}) : launch(std::false_type{}, std::false_type{});
    });
    if (rc != hipSuccess) return static_cast<int>(rc);
    j.D = a.D;
    j.param_dtype = a.param_dtype;
    j.colblocks = (a.D + kWave - 1) / kWave;
    if (a.slots > 0) {
        j.partial = a.partial;
        j.part_stride = static_cast<int64_t>(a.slots) * a.D;
        j.sum_stride = a.D;
        j.parts = p.blocks;
        hipLaunchKernelGGL(ple_norm_join_kernel, dim3(j.colblocks * a.slots), dim3(kJoinWaves * kWave), 0, r.stream, j);
    }
    if (a.gates == 2 && a.d_gate && p.pieces > 1) {
        j.partial = a.gate_partial;
        j.part_stride = a.D;
        j.sum_stride = p.pieces * a.D;
        j.parts = static_cast<int>(p.pieces);
        return static_cast<int>(join_gates(r, j));
    }
    return static_cast<int>(hipGetLastError());
}

}  // namespace ple

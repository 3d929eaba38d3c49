// Distillation from a teacher's top logits, with optional hard labels (gfx950).
// Row n has the student's logits z [V], the teacher's logits t [K] of the
// classes c [K], a temperature T and the weight alpha of the teacher:
//
//     q = softmax(z / T),  p_k = exp(t_k / T - l)
//     loss = alpha T^2 (sum_k p_k (log p_k - log q_{c_k}) + rest)
//            + (1 - alpha) (lse(z) - z[label])
//
// l is the log-sum over the row's own K logits, or is given: the log-sum over
// the teacher's whole vocabulary.  Then the mass it left out, rho = 1 - sum p,
// is one more outcome: rest = rho (log rho - log Q), Q the student's mass
// outside the K classes.  With m = sum p + rho the gradient is
//
//     dz_j = alpha T (m q_j - sum_{c_k = j} p_k - [j outside] rho q_j / Q)
//            + (1 - alpha) (softmax(z)_j - [j = label])
//
// Bound by memory: the forward reads z once, with the running maximum and the
// sums at both temperatures; the backward reads it once and writes dz once:
// every class gets the formula without its sparse terms in a dense pass, and
// the K classes and the label are then computed whole and written over it.
// With a given l the dense sums leave the K classes out, by a bit for each class
// in LDS, and their own K terms are added: Q is a sum of its own terms and not a
// difference.
//
// At T = 2 and T = 4 the exponentials of both temperatures are one: exp(x) is
// exp(x / T) squared once or twice.  (One exponential a class less, at a
// quarter of the rate of other operations.)
//
// A row belongs to a team of lanes (part of a wave, a wave or a workgroup);
// where there are few rows of many classes, to several workgroups, each a range
// of the classes, whose sums a second kernel joins.
//
// Measured (one MI355X, kernel trace): 4096 x 131072 bf16 212 us forward (5.1 TB/s
// read) and 410 backward (5.2 TB/s); 4096 x 50257 with labels at T = 2 91 and 155 us
// (4.5 and 5.3 TB/s; with two exponentials a class 125 forward); 24 x 32000 4.2 +
// 4.3 + 4.3 us and 4096 x 100 fp32 4.5 + 4.0 us, a chain of loads and joins each.
// Short rows: 262144 x 200 bf16 55 and 46 us (2.5 and 5.2 TB/s), of 100 entries a
// row 202 and 212 (2.1 and 2.5): a lane's entries are loads that follow each other.

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "ple_internal.h"
#include "ple_rows.h"

namespace ple {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct DistillArgs {
    const void *z, *t, *classes;
    const float *t_lse;          // NULL: over the row's own K logits
    const int64_t *labels;       // NULL: none
    const float *g;
    void *dz;
    float *loss;
    float *stats;                // a row: maximum, log2 of the sums at T and 1, l; m, factor outside, labelled, its base
    float *partial;              // [N, splits, 8]: maximum, sums at T and 1, whether classes occur twice and those alone
    int64_t N;
    int V, K, t_dtype, wide;     // wide: 64-bit classes
    int splits, part;            // classes a split takes
    int words;                   // of a team's bits in LDS
    float inv_t, t_factor, alpha;    // 1 / T, T
};

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ int64_t class_of(const DistillArgs &a, int64_t i) {
    return a.wide ? static_cast<const int64_t *>(a.classes)[i] : static_cast<const int32_t *>(a.classes)[i];
}

// Vectors of a row's range [c0, c1): element c0 + i is bit shift + i of the
// team's bits, so that 16-byte vectors of z own whole groups of bits.
template <int Z, bool VEC>
struct Range {
    static constexpr int kVec = VEC ? (Z == PLE_DTYPE_F32 ? 4 : 8) : 1;
    int64_t base;                // of the row
    int c0, c1, shift, head;     // head: elements before the first vector
    __device__ __forceinline__ Range(const void *z, int64_t row, int v, int begin, int end) : base(row * v), c0(begin), c1(end) {
        if constexpr (VEC) {
            shift = static_cast<int>((reinterpret_cast<uintptr_t>(z) / elem_bytes(Z) + base + begin) % kVec);
            head = min((kVec - shift) % kVec, end - begin);
        } else {
            shift = head = 0;
        }
    }
    __device__ __forceinline__ int vectors() const { return (c1 - c0 - head) / kVec; }
    __device__ __forceinline__ int at(int vec) const { return c0 + head + vec * kVec; }      // its first class
    __device__ __forceinline__ int bit(int c) const { return c - c0 + shift; }
    // classes beside the vectors: `head` before, the others behind
    __device__ __forceinline__ int odd() const { return (c1 - c0) - vectors() * kVec; }
    __device__ __forceinline__ int odd_at(int i) const { return i < head ? c0 + i : c0 + vectors() * kVec + i; }
};

// Vectors of z that a lane has in flight.
constexpr int kUnroll = 4;

// A vector of z as loaded: VEC elements of type Z.
template <int Z, int VEC>
struct Words {
    uint32_t w[grad_words<Z, VEC>()];
    __device__ __forceinline__ void load(const void *z, int64_t i) {
        if constexpr (VEC == 1) {
            if constexpr (Z == PLE_DTYPE_F32) w[0] = static_cast<const uint32_t *>(z)[i];
            else w[0] = static_cast<const uint16_t *>(z)[i];
        } else {
            const uint4 v = *reinterpret_cast<const uint4 *>(static_cast<const char *>(z) + i * elem_bytes(Z));
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        }
    }
    __device__ __forceinline__ float at(int e) const { return grad_elem<Z>(w, e); }
};

// The sums of a row: at T alone, at 1 too, or at 1 by squaring those at T.
enum { kOneSum, kTwoSums, kOneSquare, kTwoSquares };

template <int SUMS>
__device__ __forceinline__ float at_one(float x) {       // exp(v - m) from exp((v - m) / T)
    x *= x;
    return SUMS == kTwoSquares ? x * x : x;
}

// Running maximum and sums of a lane.  The maximum starts at the lowest number,
// not at -inf: a class of -inf then adds exp(-inf) = 0 without a NaN.
template <int SUMS>
struct Sums {
    float m = -FLT_MAX, at_t = 0.0f, at_1 = 0.0f;
    __device__ __forceinline__ void rescale(float to, float ct) {
        at_t *= exp2_fast((m - to) * ct);
        if constexpr (SUMS != kOneSum) at_1 *= exp2_fast((m - to) * kLog2e);
        m = to;
    }
    // adds N vectors without the classes of `skip` (bit e: element e), of which the
    // maximum is not either
    template <int N, int Z, int VEC>
    __device__ __forceinline__ void add(const Words<Z, VEC> (&w)[N], const uint32_t (&skip)[N], float ct) {
        float v[N][VEC];
#pragma unroll
        for (int k = 0; k < N; ++k) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[k][e] = w[k].at(e);
            if (skip[k])
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    if ((skip[k] >> e) & 1) v[k][e] = -__builtin_inff();
        }
        float top = v[0][0];
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) top = fmaxf(top, v[k][e]);
        if (top > m) rescale(top, ct);
        // (a sum of its own for every vector: their additions overlap)
        float part[N], part_1[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            part[k] = part_1[k] = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = v[k][e] - m, x = exp2_fast(d * ct);
                part[k] += x;
                if constexpr (SUMS == kTwoSums) part_1[k] += exp2_fast(d * kLog2e);
                else if constexpr (SUMS != kOneSum) part_1[k] += at_one<SUMS>(x);
            }
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            at_t += part[k];
            at_1 += part_1[k];
        }
    }
};

// An entry of the teacher's, or the label.
struct Entry {
    int64_t c = -1;
    float t = 0.0f, z = 0.0f;    // t / T; the student's logit (of a class in [0, V))
};

template <int Z>
__device__ __forceinline__ Entry load_entry(const DistillArgs &a, int64_t n, int k) {
    Entry e;
    if (n >= a.N || k >= a.K) return e;
    e.c = class_of(a, n * a.K + k);
    e.t = load_any(a.t, n * a.K + k, a.t_dtype) * a.inv_t;
    if (e.c >= 0 && e.c < a.V) e.z = load_grad<Z>(a.z, n * a.V + e.c);
    return e;
}

template <int Z>
__device__ __forceinline__ Entry load_label(const DistillArgs &a, int64_t n) {
    Entry e;
    if (n >= a.N || !a.labels) return e;
    e.c = a.labels[n];
    if (e.c >= 0 && e.c < a.V) e.z = load_grad<Z>(a.z, n * a.V + e.c);
    return e;
}

// Marks the row's classes of [c0, c1) in the team's bits, which it clears first;
// mine: this lane's first entry.  Returns whether one of them was there already.
template <int TEAM, int Z, bool VEC>
__device__ __forceinline__ bool mark_classes(Team<TEAM> &team, const DistillArgs &a, int64_t n, const Entry &mine,
                                             const Range<Z, VEC> &r, uint32_t *bits, int *twice) {
    for (int w = team.lane(); w < a.words; w += team.lanes()) bits[w] = 0;
    if (team.lane() == 0) *twice = 0;
    team.sync();
    if (n < a.N)
        for (int k = team.lane(); k < a.K; k += team.lanes()) {
            const int64_t c = k == team.lane() ? mine.c : class_of(a, n * a.K + k);
            if (c < r.c0 || c >= r.c1) continue;
            const int b = r.bit(static_cast<int>(c));
            if (atomicOr(&bits[b >> 5], 1u << (b & 31)) >> (b & 31) & 1) *twice = 1;
        }
    team.sync();
    return *twice != 0;
}

template <int Z, int TEAM, int SUMS>
__device__ __forceinline__ void scan_row(Team<TEAM> &team, const DistillArgs &a, const Range<Z, true> &r, const uint32_t *bits,
                                         float ct, Sums<SUMS> &s) {
    constexpr int kVec = Range<Z, true>::kVec;
    const auto inside = [&](int c, int n) -> uint32_t {
        if (!a.t_lse) return 0;
        const int b = r.bit(c);
        return bits[b >> 5] >> (b & 31) & ((1u << n) - 1);
    };
    const int vectors = r.vectors(), lanes = team.lanes();
    int i = team.lane();
    for (; i + (kUnroll - 1) * lanes < vectors; i += kUnroll * lanes) {
        Words<Z, kVec> v[kUnroll];
        uint32_t in[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) v[u].load(a.z, r.base + r.at(i + u * lanes));
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) in[u] = inside(r.at(i + u * lanes), kVec);
        s.add(v, in, ct);
    }
    for (; i < vectors; i += lanes) {
        Words<Z, kVec> v[1];
        v[0].load(a.z, r.base + r.at(i));
        const uint32_t in[1] = {inside(r.at(i), kVec)};
        s.add(v, in, ct);
    }
    for (i = team.lane(); i < r.odd(); i += lanes) {
        Words<Z, 1> v[1];
        v[0].load(a.z, r.base + r.odd_at(i));
        const uint32_t in[1] = {inside(r.odd_at(i), 1)};
        s.add(v, in, ct);
    }
}

// The marked classes alone, each once however many entries it has: by the bits,
// since an entry that looks for its class among the others makes the work the
// entries' square.
template <int Z, int TEAM, int SUMS>
__device__ __forceinline__ void scan_marked(Team<TEAM> &team, const DistillArgs &a, const Range<Z, true> &r, const uint32_t *bits,
                                            float ct, Sums<SUMS> &s) {
    for (int w = team.lane(); w < a.words; w += team.lanes())
        for (uint32_t m = bits[w]; m != 0; m &= m - 1) {
            Words<Z, 1> v[1];
            v[0].load(a.z, r.base + r.c0 + 32 * w + __builtin_ctz(m) - r.shift);
            const uint32_t in[1] = {0};
            s.add(v, in, ct);
        }
}

// The row's loss and stats from its lanes' sums.  mine: this lane's first entry.
// With a given l the sums and their maximum leave out the K classes: the outside
// mass keeps its own scale, however far below the row's maximum it is.  named(): this
// lane's sums of the K classes where one of them occurs `twice`.
template <int Z, int TEAM, int SUMS, typename Named>
__device__ __forceinline__ void finish_row(Team<TEAM> &team, const DistillArgs &a, int64_t n, const Entry &mine,
                                           const Entry &label, Sums<SUMS> &s, bool twice, Named named) {
    const bool on = n < a.N, tail = a.t_lse != nullptr;
    const float ct = a.inv_t * kLog2e;
    const auto each = [&](auto f) {
        for (int k = team.lane(); on && k < a.K; k += team.lanes()) f(k, k == team.lane() ? mine : load_entry<Z>(a, n, k));
    };
    const auto in_range = [&](const Entry &e) { return e.c >= 0 && e.c < a.V; };
    float top[2] = {s.m, -FLT_MAX};      // of the sums; of the K classes (given l), else the teacher's
    each([&](int, const Entry &e) {
        if (tail ? in_range(e) : e.c >= 0) top[1] = fmaxf(top[1], tail ? e.z : e.t);
    });
    team.maxima(top);
    s.rescale(top[0], ct);
    const float peak = tail ? fmaxf(s.m, top[1]) : s.m;
    // sums: at T, at 1; of the K classes at T, at 1 (given l), else the teacher's; its
    // mass and cross terms (given l); entries, with 2^12 for one beyond V
    enum { kSumT, kSum1, kInT, kIn1, kMassP, kCross, kCount, kValues };
    constexpr float kWrong = 4096.0f;
    float v[kValues] = {s.at_t, s.at_1, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    float lse = tail && on ? a.t_lse[n] : 0.0f;
    bool some = false, wrong = false;
    each([&](int, const Entry &e) {
        if (e.c < 0) return;
        some = true;
        wrong = wrong || e.c >= a.V;
        if (!tail) {
            v[kInT] += exp2_fast((e.t - top[1]) * kLog2e);
            return;
        }
        if (!in_range(e)) return;
        v[kInT] += exp2_fast((e.z - peak) * ct);
        v[kIn1] += exp2_fast((e.z - peak) * kLog2e);
        const float log_p = e.t - lse, p = exp2_fast(log_p * kLog2e);
        v[kMassP] += p;
        if (p != 0.0f) v[kCross] += p * (log_p - (e.z - peak) * a.inv_t);
    });
    if (__builtin_expect(twice, 0)) {
        Sums<SUMS> once = named();
        once.rescale(peak, ct);
        v[kInT] = once.at_t;
        v[kIn1] = once.at_1;
    }
    v[kCount] = (some ? 1.0f : 0.0f) + (wrong ? kWrong : 0.0f);      // (exact: at most 256 lanes)
    team.sums(v);
    bool taught = v[kCount] != 0.0f;
    wrong = v[kCount] >= kWrong;
    const float outside = v[kSumT];
    float at_t = outside, at_1 = SUMS == kOneSum ? v[kSumT] : v[kSum1], kd = v[kCross], mass = v[kMassP];
    const float down = tail ? exp2_fast((s.m - peak) * ct) : 1.0f;       // from the sums' scale to the row's
    if (tail) {
        at_t = outside * down + v[kInT];
        at_1 = SUMS == kOneSum ? at_t : at_1 * exp2_fast((s.m - peak) * kLog2e) + v[kIn1];
    }
    const float log_t = logf(at_t), log_1 = logf(at_1);
    if (tail) {
        kd += mass * log_t;
    } else {
        if (v[kInT] == 0.0f) taught = false;     // (no class has a probability)
        lse = taught ? top[1] + logf(v[kInT]) : 0.0f;
        each([&](int, const Entry &e) {
            if (!in_range(e)) return;
            const float log_p = e.t - lse, p = exp2_fast(log_p * kLog2e);
            mass += p;
            if (p != 0.0f) kd += p * (log_p - (e.z - peak) * a.inv_t + log_t);
        });
        team.sum2(kd, mass);
    }
    if (team.lane() != 0 || !on) return;
    // factor: what a class without sparse terms has its exp((z - base) / T) times
    float factor = mass / at_t, base = peak, labelled = 0.0f, ce = 0.0f, m = peak;
    if (tail && taught) {
        const float rho = fmaxf(1.0f - mass, 0.0f), gap = (s.m - peak) * a.inv_t;
        // (a row whose K classes are all there are has no outside; nor has one whose
        // others are at the type's lowest value: a mass below what 64 bits hold is none)
        if (rho > 0.0f && outside > 0.0f && gap > -700.0f) {
            kd += rho * (logf(rho) - (logf(outside) + gap) + log_t);
            mass += rho;
            factor = mass * down / at_t - rho / outside;
            base = s.m;
        }
    }
    if (label.c >= a.V) labelled = ce = __builtin_nanf("");
    else if (label.c >= 0) {
        labelled = 1.0f;
        ce = log_1 - (label.z - m);
    }
    if (wrong) kd = mass = factor = __builtin_nanf("");
    const bool live = at_t != 0.0f;      // else every class is masked: no loss, no gradient
    if (!live) kd = ce = m = mass = factor = base = labelled = 0.0f;
    float4 *st = reinterpret_cast<float4 *>(a.stats + n * PLE_DISTILL_STATS);
    st[0] = make_float4(m, live ? log_t * kLog2e : 0.0f, live ? log_1 * kLog2e : 0.0f, lse);
    st[1] = make_float4(mass, factor, labelled, base);
    a.loss[n] = (a.alpha > 0.0f && taught ? a.alpha * a.t_factor * a.t_factor * kd : 0.0f) +
                (a.alpha < 1.0f && labelled != 0.0f ? (1.0f - a.alpha) * ce : 0.0f);
}

template <int Z, int TEAM, int SUMS>
__global__ __launch_bounds__(Team<TEAM>::kThreads) void ple_distill_forward_kernel(DistillArgs a) {
    extern __shared__ uint32_t s_bits[];
    __shared__ float s_sum[Team<TEAM>::kLdsFloats];
    __shared__ int s_twice[Team<TEAM>::kThreads / (TEAM < kBlock ? TEAM : kBlock)];
    Team<TEAM> team(s_sum);
    const int splits = TEAM < kBlock ? 1 : a.splits, split = blockIdx.x % splits;    // (only workgroups' rows are split)
    const int64_t n = static_cast<int64_t>(blockIdx.x / splits) * team.per_block() + team.index();
    const float ct = a.inv_t * kLog2e;
    uint32_t *bits = s_bits + team.index() * a.words;
    const Range<Z, true> r(a.z, n, a.V, split * a.part, min(a.V, (split + 1) * a.part));
    const Entry mine = load_entry<Z>(a, n, team.lane()), label = load_label<Z>(a, n);
    Sums<SUMS> s;
    const bool twice = a.t_lse && mark_classes(team, a, n, mine, r, bits, &s_twice[team.index()]);
    if (n < a.N) scan_row<Z, TEAM, SUMS>(team, a, r, bits, ct, s);
    const auto marked = [&] {        // (none where n is past the rows)
        Sums<SUMS> v;
        scan_marked(team, a, r, bits, ct, v);
        return v;
    };
    if (splits == 1) {
        finish_row<Z>(team, a, n, mine, label, s, twice, marked);
        return;
    }
    const auto join = [&](Sums<SUMS> &v) {
        float top[1] = {v.m};
        team.maxima(top);
        v.rescale(top[0], ct);
        team.sum2(v.at_t, v.at_1);
    };
    join(s);
    const bool out = team.lane() == 0 && n < a.N;
    float4 *part = reinterpret_cast<float4 *>(a.partial) + 2 * (n * splits + split);
    if (out) part[0] = make_float4(s.m, s.at_t, s.at_1, twice ? 1.0f : 0.0f);
    if (__builtin_expect(twice, 0)) {
        Sums<SUMS> v = marked();
        join(v);
        if (out) part[1] = make_float4(v.m, v.at_t, v.at_1, 0.0f);
    }
}

// A row's sums from its splits' (one wave a row), then its loss.
template <int Z, int SUMS>
__global__ __launch_bounds__(kBlock) void ple_distill_join_kernel(DistillArgs a) {
    Team<kWave> team(nullptr);
    const int64_t n = static_cast<int64_t>(blockIdx.x) * team.per_block() + team.index();
    const Entry mine = load_entry<Z>(a, n, team.lane()), label = load_label<Z>(a, n);
    Sums<SUMS> s;
    const float4 *parts = reinterpret_cast<const float4 *>(a.partial) + 2 * n * a.splits;
    const auto add = [&](Sums<SUMS> &to, const float4 &v) {
        Sums<SUMS> part;
        part.m = v.x;
        part.at_t = v.y;
        part.at_1 = v.z;
        const float top = fmaxf(to.m, part.m);
        to.rescale(top, a.inv_t * kLog2e);
        part.rescale(top, a.inv_t * kLog2e);
        to.at_t += part.at_t;
        to.at_1 += part.at_1;
    };
    bool twice = false;
    for (int i = team.lane(); n < a.N && i < a.splits; i += kWave) {
        const float4 v = parts[2 * i];
        add(s, v);
        twice = twice || v.w != 0.0f;
    }
    // the splits where a class occurs twice have their own sums, the others' entries are all there is
    const auto named = [&] {
        Sums<SUMS> v;
        for (int i = team.lane(); i < a.splits; i += kWave)
            if (parts[2 * i].w != 0.0f) add(v, parts[2 * i + 1]);
        for (int k = team.lane(); k < a.K; k += kWave) {
            const Entry e = load_entry<Z>(a, n, k);
            if (e.c >= 0 && e.c < a.V && parts[2 * (static_cast<int>(e.c) / a.part)].w == 0.0f)
                add(v, make_float4(e.z, 1.0f, 1.0f, 0.0f));
        }
        return v;
    };
    finish_row<Z>(team, a, n, mine, label, s, __any(twice), named);
}

// Entries of a row with repeats up to which each looks through them all for its class's
// others; beyond, that is their square, and sum_repeats takes them (backwards of rows
// with a repeat, searched / by sum_repeats: 512 x 50257 of 512 entries 230 / 307 us, of
// 1024 800 / 546; 4096 x 2000 of 128 85 / 115, of 256 270 / 213; 16384 x 100 of 64 67 /
// 103, of 128 314 / 240, of 2048 134 / 6.8 ms).
template <int TEAM>
constexpr int kSearched = 64 + 2 * TEAM;

// put(entry, sum of its class's probabilities) for every entry in [c0, c1): as many
// classes at a time as the team's bits have room for sums of (the bits are lost), to
// which one wave adds the entries in their own order.
template <int TEAM, int Z, bool VEC, typename Prob, typename Put>
__device__ __forceinline__ void sum_repeats(Team<TEAM> &team, const DistillArgs &a, int64_t n, const Range<Z, VEC> &r,
                                            uint32_t *bits, Prob prob, Put put) {
    constexpr int kLanes = TEAM < kWave ? TEAM : kWave;
    volatile float *sums = reinterpret_cast<volatile float *>(bits);
    const int first = threadIdx.x % kWave / kLanes * kLanes;     // of the team in its wave
    for (int lo = r.c0; lo < r.c1; lo += a.words) {
        const int hi = min(lo + a.words, r.c1);
        for (int w = team.lane(); w < a.words; w += team.lanes()) sums[w] = 0.0f;
        team.sync();
        for (int k0 = 0; team.lane() < kLanes && k0 < a.K; k0 += kLanes) {
            const int k = k0 + team.lane();
            const int64_t c = k < a.K ? class_of(a, n * a.K + k) : -1;
            const bool on = c >= lo && c < hi;
            const float p = on ? prob(load_any(a.t, n * a.K + k, a.t_dtype) * a.inv_t) : 0.0f;
            for (uint64_t todo = __ballot(on) >> first & (~uint64_t{0} >> (kWave - kLanes)); todo != 0; todo &= todo - 1) {
                if (team.lane() == __builtin_ctzll(todo)) sums[c - lo] = sums[c - lo] + p;
                __builtin_amdgcn_wave_barrier();
            }
        }
        team.sync();
        for (int k = team.lane(); k < a.K; k += team.lanes()) {
            const Entry e = load_entry<Z>(a, n, k);
            if (e.c >= lo && e.c < hi) put(e, sums[e.c - lo]);
        }
        team.sync();
    }
}

template <int Z, int TEAM, bool VEC, int SUMS, bool NT>
__global__ __launch_bounds__(Team<TEAM>::kThreads) void ple_distill_backward_kernel(DistillArgs a) {
    constexpr int kVec = Range<Z, VEC>::kVec;
    extern __shared__ uint32_t s_bits[];
    __shared__ int s_twice[Team<TEAM>::kThreads / (TEAM < kBlock ? TEAM : kBlock)];
    Team<TEAM> team(nullptr);
    // the last rows first: the forward left them in the memory-side cache
    const unsigned block = gridDim.x - 1 - blockIdx.x;
    const int splits = TEAM < kBlock ? 1 : a.splits, split = block % splits;
    const int64_t n = static_cast<int64_t>(block / splits) * team.per_block() + team.index();
    const float ct = a.inv_t * kLog2e;
    uint32_t *bits = s_bits + team.index() * a.words;
    const Range<Z, VEC> r(a.z, n, a.V, split * a.part, min(a.V, (split + 1) * a.part));
    const Entry mine = load_entry<Z>(a, n, team.lane());
    Entry label = load_label<Z>(a, n);
    float4 st0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), st1 = st0;
    float g = 0.0f;
    if (n < a.N) {
        const float4 *st = reinterpret_cast<const float4 *>(a.stats + n * PLE_DISTILL_STATS);
        st0 = st[0];
        st1 = st[1];
        g = a.g[n];
    }
    const bool twice = mark_classes(team, a, n, mine, r, bits, &s_twice[team.index()]);
    const float peak = st0.x, log_t = st0.y, log_1 = st0.z, lse = st0.w, mass = st1.x, base = st1.w;
    const float w_soft = a.alpha > 0.0f && mass != 0.0f ? g * a.alpha * a.t_factor : 0.0f;
    const float w_out = w_soft != 0.0f ? w_soft * st1.y : 0.0f;
    const float w_hard = a.alpha < 1.0f && st1.z != 0.0f ? g * (1.0f - a.alpha) * st1.z : 0.0f;
    if (st1.z == 0.0f) label.c = -1;
    const auto soft = [&](float z) { return exp2_fast((z - peak) * ct - log_t); };
    const auto hard = [&](float z) { return exp2_fast((z - peak) * kLog2e - log_1); };
    // The dense terms, from the outside classes' own scale; of the K classes they may
    // overflow, and are written over.
    const float w_1 = w_hard * exp2_fast((base - peak) * kLog2e - log_1), w_t = SUMS == kOneSum ? w_out + w_1 : w_out;
    const auto dense = [&](float z) {
        const float d = z - base, x = exp2_fast(d * ct);
        if constexpr (SUMS == kOneSum) return w_t * x;
        else if constexpr (SUMS == kTwoSums) return w_t * x + w_1 * exp2_fast(d * kLog2e);
        else return w_t * x + w_1 * at_one<SUMS>(x);
    };
    if (n < a.N) {
        const int vectors = r.vectors(), lanes = team.lanes();
        const auto put = [&](const Words<Z, kVec> &w, int64_t at) {
            float v[kVec];
#pragma unroll
            for (int e = 0; e < kVec; ++e) v[e] = dense(w.at(e));
            store_vec<Z, kVec, NT>(a.dz, at, v);
        };
        int i = team.lane();
        for (; i + (kUnroll - 1) * lanes < vectors; i += kUnroll * lanes) {
            Words<Z, kVec> w[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) w[u].load(a.z, r.base + r.at(i + u * lanes));
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) put(w[u], r.base + r.at(i + u * lanes));
        }
        for (; i < vectors; i += lanes) {
            Words<Z, kVec> w;
            w.load(a.z, r.base + r.at(i));
            put(w, r.base + r.at(i));
        }
        if constexpr (VEC)
            for (int i = team.lane(); i < r.odd(); i += team.lanes()) {
                const float v = dense(load_grad<Z>(a.z, r.base + r.odd_at(i)));
                store_vec<Z, 1>(a.dz, r.base + r.odd_at(i), &v);
            }
    }
    team.sync();
    if (n >= a.N) return;
    const auto prob = [&](float t) { return exp2_fast((t - lse) * kLog2e); };
    const auto put = [&](const Entry &e, float p) {
        float v = w_soft != 0.0f ? w_soft * (mass * soft(e.z) - p) : 0.0f;
        if (w_hard != 0.0f) v += w_hard * (hard(e.z) - (e.c == label.c ? 1.0f : 0.0f));
        store_vec<Z, 1>(a.dz, r.base + e.c, &v);
    };
    if (team.lane() == 0 && label.c >= r.c0 && label.c < r.c1) {
        const int b = r.bit(static_cast<int>(label.c));
        if (!(bits[b >> 5] >> (b & 31) & 1)) {
            const float v = dense(label.z) - w_hard;
            store_vec<Z, 1>(a.dz, r.base + label.c, &v);
        }
    }
    if (__builtin_expect(twice && a.K > kSearched<TEAM>, 0)) {
        team.sync();         // (the label's bit is read)
        sum_repeats(team, a, n, r, bits, prob, put);
        return;
    }
    for (int k = team.lane(); k < a.K; k += team.lanes()) {
        const Entry e = k == team.lane() ? mine : load_entry<Z>(a, n, k);
        if (e.c < r.c0 || e.c >= r.c1) continue;
        float p = 0.0f;
        bool first = true;
        if (twice) {
            for (int i = 0; i < a.K; ++i)
                if (class_of(a, n * a.K + i) == e.c) {
                    first = first && i >= k;
                    p += prob(load_any(a.t, n * a.K + i, a.t_dtype) * a.inv_t);
                }
        } else {
            p = prob(e.t);
        }
        if (first) put(e, p);
    }
}

// ---------------------------------------------------------------------------
// plans and launches
// ---------------------------------------------------------------------------

struct DistillPlan {
    int team, threads, per_block, splits, part, words;
    size_t bytes, lds;
};

constexpr int kMaxPart = 1 << 18;        // classes a workgroup has bits for, about (32 KB)

DistillPlan plan_distill(int64_t N, int64_t V, int vec = 8) {
    // Lanes a row: a few vectors for each, of `vec` classes (65536 rows, both ways: 200
    // classes bf16 by waves 80 us, by 16 lanes 34; 500 87 and 72; 500 fp32, 125 vectors,
    // 96 and 104), a workgroup beyond 4096 classes (bf16: 16384 x 2100 by workgroups 91
    // us, by waves 50; x 4096 100 and 75; 8192 x 8192 76 and 74).
    // Splits: four workgroups a CU where the rows are fewer, 2048 classes each at
    // least.
    DistillPlan p{};
    p.team = V <= 8 * vec ? 8 : (V <= 64 * vec ? 16 : (V <= 4096 ? kWave : kBlock));
    p.threads = kBlock;
    p.per_block = kBlock / p.team;
    p.splits = 1;
    p.part = static_cast<int>(V);
    if (p.team == kBlock) {
        const int64_t wanted = std::max<int64_t>((4 * device_cu_count() + N - 1) / std::max<int64_t>(N, 1), (V + kMaxPart - 1) / kMaxPart);
        const int64_t splits = std::max((V + kMaxPart - 1) / kMaxPart, std::min(wanted, V / 2048));
        if (splits > 1) {
            p.part = static_cast<int>(((V + splits - 1) / splits + 63) / 64 * 64);
            p.splits = static_cast<int>((V + p.part - 1) / p.part);
        }
    }
    p.words = (p.part + 8 + 31) / 32;
    p.lds = static_cast<size_t>(p.words) * 4 * p.per_block;
    p.bytes = p.splits > 1 ? align_up(static_cast<size_t>(N) * p.splits * 32, 256) : 0;
    return p;
}

DistillArgs distill_args(const DistillRequest &r, const DistillPlan &p) {
    DistillArgs a{};
    a.z = r.logits; a.t = r.teacher; a.classes = r.classes;
    a.t_lse = r.teacher_lse; a.labels = r.labels;
    a.g = r.g; a.dz = r.dz; a.loss = r.loss; a.stats = r.stats;
    a.partial = static_cast<float *>(r.workspace);
    a.N = r.N; a.V = static_cast<int>(r.V); a.K = static_cast<int>(r.K);
    a.t_dtype = r.teacher_dtype; a.wide = r.wide;
    a.splits = p.splits; a.part = p.part; a.words = p.words;
    a.inv_t = 1.0f / r.temperature; a.t_factor = r.temperature; a.alpha = r.alpha;
    return a;
}

// f(type, team, sums) as compile-time constants
template <typename F>
hipError_t with_distill(const DistillRequest &r, const DistillPlan &p, F f) {
    const auto by_sums = [&](auto z, auto team) {
        if (!r.labels || r.temperature == 1.0f) return f(z, team, std::integral_constant<int, kOneSum>{});
        if (r.temperature == 2.0f) return f(z, team, std::integral_constant<int, kOneSquare>{});
        if (r.temperature == 4.0f) return f(z, team, std::integral_constant<int, kTwoSquares>{});
        return f(z, team, std::integral_constant<int, kTwoSums>{});
    };
    const auto by_team = [&](auto z) {
        switch (p.team) {
            case 8: return by_sums(z, std::integral_constant<int, 8>{});
            case 16: return by_sums(z, std::integral_constant<int, 16>{});
            case kWave: return by_sums(z, std::integral_constant<int, kWave>{});
            default: return by_sums(z, std::integral_constant<int, kBlock>{});
        }
    };
    switch (r.dtype) {
        case PLE_DTYPE_F32: return by_team(std::integral_constant<int, PLE_DTYPE_F32>{});
        case PLE_DTYPE_F16: return by_team(std::integral_constant<int, PLE_DTYPE_F16>{});
        default: return by_team(std::integral_constant<int, PLE_DTYPE_BF16>{});
    }
}

constexpr int64_t kMaxBlocks = 1 << 23;  // of a launch: a grid holds fewer than 2^32 threads

// f(arguments, grid) for the rows of one launch after another.
template <typename F>
hipError_t for_rows(const DistillRequest &r, const DistillPlan &p, const DistillArgs &a, F f) {
    const int64_t most = std::max<int64_t>(1, kMaxBlocks / p.splits) * p.per_block;
    for (int64_t n = 0; n < r.N; n += most) {
        DistillArgs b = a;
        const auto skip = [n](auto *&q, int64_t elems, int bytes) {
            if (q) q = reinterpret_cast<std::remove_reference_t<decltype(q)>>(reinterpret_cast<uintptr_t>(q) + n * elems * bytes);
        };
        b.N = std::min(most, r.N - n);
        skip(b.z, r.V, elem_bytes(r.dtype));
        skip(b.dz, r.V, elem_bytes(r.dtype));
        skip(b.t, r.K, elem_bytes(r.teacher_dtype));
        skip(b.classes, r.K, r.wide ? 8 : 4);
        skip(b.t_lse, 1, 4);
        skip(b.labels, 1, 8);
        skip(b.g, 1, 4);
        skip(b.loss, 1, 4);
        skip(b.stats, PLE_DISTILL_STATS, 4);
        skip(b.partial, 8 * p.splits, 4);
        const hipError_t rc = f(b, dim3(static_cast<unsigned>((b.N + p.per_block - 1) / p.per_block * p.splits)));
        if (rc != hipSuccess) return rc;
    }
    return hipSuccess;
}

}  // namespace

// (rows that are split are a workgroup's whatever the type)
size_t distill_workspace_bytes(int64_t N, int64_t V) { return plan_distill(N, V).bytes; }

int distill_run(const DistillRequest &r) {
    const DistillPlan p = plan_distill(r.N, r.V, 16 / elem_bytes(r.dtype));
    if (p.bytes > 0 && (!r.workspace || r.workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(r.workspace) % 256 != 0))
        return PLE_E_WORKSPACE;
    return static_cast<int>(for_rows(r, p, distill_args(r, p), [&](const DistillArgs &a, dim3 grid) {
        const hipError_t rc = with_distill(r, p, [&](auto z, auto team, auto sums) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_distill_forward_kernel<decltype(z)::value, decltype(team)::value,
                                                                          decltype(sums)::value>),
                               grid, dim3(p.threads), p.lds, r.stream, a);
            return hipGetLastError();
        });
        if (rc != hipSuccess || p.splits == 1) return rc;
        const dim3 rows(static_cast<unsigned>((a.N + kWavesPerBlock - 1) / kWavesPerBlock));
        return with_distill(r, p, [&](auto z, auto, auto sums) {
            hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_distill_join_kernel<decltype(z)::value, decltype(sums)::value>), rows,
                               dim3(kBlock), 0, r.stream, a);
            return hipGetLastError();
        });
    }));
}

int distill_backward_run(const DistillRequest &r) {
    const DistillPlan p = plan_distill(r.N, r.V, 16 / elem_bytes(r.dtype));
    // One vector for z and dz: both addresses are the same way into 16 bytes.  Else an
    // element at a time: most row slices of logits of odd widths (4096 x 50257 bf16
    // 182 -> 218 us, 65536 x 2101 120 -> 145).
    const bool vec = (reinterpret_cast<uintptr_t>(r.logits) - reinterpret_cast<uintptr_t>(r.dz)) % 16 == 0;
    // Long rows' gradients of 64 MB on are stored past the caches, which the logits
    // need (50257 classes, both kernels: 2560 rows 178 -> 145 us, 1024 73 -> 62, 512
    // and fewer as fast either way; short rows, of parts of lines, are 3 to 5%
    // slower so at any size).
    const bool stream = p.team == kBlock && r.N * r.V * elem_bytes(r.dtype) >= (int64_t{64} << 20);
    return static_cast<int>(for_rows(r, p, distill_args(r, p), [&](const DistillArgs &a, dim3 grid) {
        return with_distill(r, p, [&](auto z, auto team, auto sums) {
            const auto launch = [&](auto v, auto nt) {
                hipLaunchKernelGGL(HIP_KERNEL_NAME(ple_distill_backward_kernel<decltype(z)::value, decltype(team)::value,
                                                                               decltype(v)::value, decltype(sums)::value,
                                                                               decltype(nt)::value>),
                                   grid, dim3(p.threads), p.lds, r.stream, a);
                return hipGetLastError();
            };
            if (!vec) return launch(std::false_type{}, std::false_type{});
            if constexpr (decltype(team)::value == kBlock)
                if (stream) return launch(std::true_type{}, std::true_type{});
            return launch(std::true_type{}, std::false_type{});
        });
    }));
}

}  // namespace ple

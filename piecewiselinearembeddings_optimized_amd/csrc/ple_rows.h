// Device-side helpers of the row operators (lookup, residual norm,
// distillation loss): element vectors of any of the three types, parameters
// whose type is known at run time, and sums over the lanes that share a row.
#pragma once

#include "ple_device.h"

namespace ple {

__host__ __device__ constexpr int elem_bytes(int dtype) { return dtype == PLE_DTYPE_F32 ? 4 : 2; }

// VEC consecutive elements of type T from element i (aligned for the access:
// VEC elements, 16 bytes at most), as floats.  VEC in {1, 2, 4, 8}.
template <int T, int VEC>
__device__ __forceinline__ void load_vec(const void *p, int64_t i, float *v) {
    load_grad_vec<T, VEC>(p, i, v);
}

// VEC consecutive floats rounded to type T and stored from element i.  NT: past
// the caches.
template <int T, int VEC, bool NT = false>
__device__ __forceinline__ void store_vec(void *p, int64_t i, const float *v) {
    if constexpr (T == PLE_DTYPE_F32 && VEC == 8) {
        store_out<T, 4, NT>(p, i, v);
        store_out<T, 4, NT>(p, i + 4, v + 4);
    } else {
        store_out<T, VEC, NT>(p, i, v);
    }
}

// One element of a type known at run time (the same for the whole launch).
__device__ __forceinline__ float load_any(const void *p, int64_t i, int dtype) {
    if (dtype == PLE_DTYPE_F32) return static_cast<const float *>(p)[i];
    const uint16_t h = static_cast<const uint16_t *>(p)[i];
    return dtype == PLE_DTYPE_BF16 ? bf16_to_float(h) : f16_to_float(h);
}

__device__ __forceinline__ void store_any(void *p, int64_t i, float v, int dtype) {
    if (dtype == PLE_DTYPE_F32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = dtype == PLE_DTYPE_BF16 ? bf16_bits(v) : f16_bits(v);
}

// Maximum over aligned groups of W lanes (a power of two), to all of them; NaN is
// passed over.  As group_sum.
template <int W>
__device__ __forceinline__ float group_max(float v) {
    if constexpr (W >= 2) v = fmaxf(v, dpp_f32<0xB1>(v));
    if constexpr (W >= 4) v = fmaxf(v, dpp_f32<0x4E>(v));
    if constexpr (W >= 8) v = fmaxf(v, dpp_f32<0x141>(v));
    if constexpr (W >= 16) v = fmaxf(v, dpp_f32<0x140>(v));
    if constexpr (W >= 32) v = fmaxf(v, __shfl_xor(v, 16));
    if constexpr (W >= 64) v = fmaxf(v, __shfl_xor(v, 32));
    return v;
}

// The lanes that share a row.  TEAM: 8, 16, 32 or 64 lanes inside a wave, or
// (more than 64) a workgroup of at most that many threads.
template <int TEAM>
struct Team {
    static constexpr bool kBlockWide = TEAM > kWave;
    static constexpr int kThreads = kBlockWide ? TEAM : kBlock;
    static constexpr int kWaves = !kBlockWide ? 1 : TEAM <= 256 ? 4 : TEAM <= 512 ? 8 : 16;      // at most
    static constexpr int kMost = 8;              // values of one sum or maximum
    static constexpr int kLdsFloats = kBlockWide ? 2 * kMost * kWaves : 1;
    float *lds;                  // kLdsFloats floats
    int turn = 0;
    __device__ __forceinline__ explicit Team(float *s) : lds(s) {}
    __device__ __forceinline__ int lane() const { return kBlockWide ? threadIdx.x : threadIdx.x % TEAM; }
    __device__ __forceinline__ int lanes() const { return kBlockWide ? blockDim.x : TEAM; }
    __device__ __forceinline__ int index() const { return kBlockWide ? 0 : threadIdx.x / TEAM; }
    __device__ __forceinline__ int per_block() const { return kBlockWide ? 1 : kBlock / TEAM; }

    // Orders the team's LDS and global accesses before it with those after it.
    __device__ __forceinline__ void sync() const {
        if constexpr (kBlockWide) {
            __syncthreads();
        } else {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    }

    // N values of each wave to all lanes, a wave's a lane (`none` past the last):
    // every aligned group of kWaves lanes has them all, to be joined by DPP
    template <int N>
    __device__ __forceinline__ void spread(float (&v)[N], float none) {
        static_assert(N <= kMost, "values");
        // (two buffers in turn: a wave can be one ahead of another)
        float *buf = lds + (turn ^= 1) * (kMost * kWaves);
        if (threadIdx.x % kWave == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) buf[threadIdx.x / kWave * N + i] = v[i];
        __syncthreads();
        const int w = threadIdx.x % kWaves;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = w < static_cast<int>(blockDim.x) / kWave ? buf[w * N + i] : none;
    }
    // sums of N values over the team's lanes, to all of them
    template <int N>
    __device__ __forceinline__ void sums(float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = group_sum<kBlockWide ? kWave : TEAM>(v[i]);
        if constexpr (kBlockWide) {
            spread(v, 0.0f);
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = group_sum<kWaves>(v[i]);
        }
    }
    __device__ __forceinline__ void sum2(float &a, float &b) {
        float v[2] = {a, b};
        sums(v);
        a = v[0];
        b = v[1];
    }
    __device__ __forceinline__ float sum(float a) {
        float v[1] = {a};
        sums(v);
        return v[0];
    }
    // maxima (NaN is passed over), to all lanes
    template <int N>
    __device__ __forceinline__ void maxima(float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = group_max<kBlockWide ? kWave : TEAM>(v[i]);
        if constexpr (kBlockWide) {
            spread(v, -__builtin_inff());
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = group_max<kWaves>(v[i]);
        }
    }
};

}  // namespace ple

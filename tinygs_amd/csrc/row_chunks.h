// Rows held in the registers of the lanes that share them, in chunks of 16 bytes
// each: what the norms' kernels load, store and sum.
#pragma once

#include "network.h"

namespace tgs {

template <class T>
constexpr int kChunk = 16 / (int)sizeof(T);

template <class T>
struct ChunkOf {
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// Chunk `c` of a row of n elements as floats; elements past the row are 0.
template <class T>
__device__ __forceinline__ void load_chunk(const T* row, int c, int n, float* v) {
    constexpr int V = kChunk<T>;
    if ((c + 1) * V <= n) {
        const auto u = *(const typename ChunkOf<T>::type*)(row + c * V);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (float)u[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = c * V + i < n ? (float)row[c * V + i] : 0.0f;
    }
}

template <class T>
__device__ __forceinline__ void store_chunk(T* row, int c, int n, const float* v) {
    constexpr int V = kChunk<T>;
    if ((c + 1) * V <= n) {
        typename ChunkOf<T>::type u;
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = (T)v[i];
        *(typename ChunkOf<T>::type*)(row + c * V) = u;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c * V + i < n) row[c * V + i] = (T)v[i];
    }
}

// A vector's chunk; `otherwise` past the end or where there is no vector.
template <int V>
__device__ __forceinline__ void load_vector(const float* p, int c, int n, float otherwise, float* v) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = p && c * V + i < n ? p[c * V + i] : otherwise;
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}

// Sums of N values over the group's lanes, the same bits in each of them.
// Within a wave: butterflies over quads, rows of 8 and 16 lanes (DPP), halves
// and the wave (lane swaps). A workgroup joins its waves' sums through LDS, in
// the order of the waves; `s` alternates between two places from call to call,
// so that one barrier a call is enough.
template <int LANES, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* s, int& turn) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        float x = v[k];
        if constexpr (LANES >= 2) x = dpp_add<0xB1>(x);     // lane ^ 1
        if constexpr (LANES >= 4) x = dpp_add<0x4E>(x);     // lane ^ 2
        if constexpr (LANES >= 8) x = dpp_add<0x141>(x);    // mirrored in 8 lanes
        if constexpr (LANES >= 16) x = dpp_add<0x140>(x);   // mirrored in 16 lanes
        if constexpr (LANES >= 32) {
            const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x),
                                                            __builtin_bit_cast(uint32_t, x), false, false);
            x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
        }
        if constexpr (LANES >= 64) {
            const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x),
                                                            __builtin_bit_cast(uint32_t, x), false, false);
            x = __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
        }
        v[k] = x;
    }
    if constexpr (LANES > 64) {
        constexpr int kWaves = LANES / 64;
        float* at = s + turn * kWaves * N;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) at[(threadIdx.x >> 6) * N + k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            float x = at[k];
            for (int w = 1; w < kWaves; ++w) x += at[w * N + k];
            v[k] = x;
        }
    }
}

}  // namespace tgs

// rows.h — device helpers of the row operators (residual joins, distillation, 4-bit layers):
// vectors of a row's elements whatever the row's width, and sums over the threads of a row.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_math.h"

namespace skl {

// A vector of V elements of T that may sit at any multiple of sizeof(T): global memory takes a
// vector at any address.
template <typename T, int V> struct Unaligned {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};

// Elements [i, i + V) of p as floats; those from `end` on read as `fill` and are not touched.
template <typename T, int V>
__device__ __forceinline__ void load_row(const void *p, uint32_t i, uint32_t end, float (&v)[V], float fill = 0.0f) {
    const T *q = reinterpret_cast<const T *>(p);
    if (i + V <= end) {
        const auto w = *reinterpret_cast<const typename Unaligned<T, V>::type *>(q + i);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (float)w[e];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = i + e < end ? (float)q[i + e] : fill;
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_row(void *p, uint32_t i, uint32_t end, const float (&v)[V]) {
    T *q = reinterpret_cast<T *>(p);
    if (i + V <= end) {
        typename Unaligned<T, V>::type w;
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = (T)v[e];
        *reinterpret_cast<typename Unaligned<T, V>::type *>(q + i) = w;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (i + e < end) q[i + e] = (T)v[e];
    }
}

// v combined over groups of 16 lanes, or over all 64 (which are then active), the same in each of
// them, in one order: by DPP, a VALU modifier, where a shuffle would go through LDS each time.
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_of(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
template <int LANES, class Op> __device__ __forceinline__ float lanes_all(float v, Op op) {
    static_assert(LANES == 16 || LANES == 64, "a DPP row or a wave");
    v = op(v, dpp<0xB1>(v));    // quad_perm 1 0 3 2
    v = op(v, dpp<0x4E>(v));    // quad_perm 2 3 0 1
    v = op(v, dpp<0x141>(v));   // row_half_mirror
    v = op(v, dpp<0x140>(v));   // row_mirror
    if constexpr (LANES == 64) v = op(op(lane_of(v, 0), lane_of(v, 16)), op(lane_of(v, 32), lane_of(v, 48)));
    return v;
}
template <int LANES = 64> __device__ __forceinline__ float lanes_sum(float v) {
    return lanes_all<LANES>(v, [](float a, float b) { return a + b; });
}
template <int LANES = 64> __device__ __forceinline__ float lanes_max(float v) {
    return lanes_all<LANES>(v, [](float a, float b) { return fmaxf(a, b); });
}

// The sum of v over the NT threads of a row, in every one of them, in a fixed order.  slot: NT / 64
// floats of LDS that no other sum uses until every thread has passed another barrier.
template <int NT> __device__ __forceinline__ float row_sum(float v, float *slot) {
    v = lanes_sum(v);
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63u) == 0) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) v += slot[w];
    }
    return v;
}

}  // namespace skl

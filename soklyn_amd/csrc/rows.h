// rows.h — device helpers of the row operators (residual joins, distillation, 4-bit layers):
// V consecutive elements at any element alignment, and sums over the threads of a row.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_math.h"

namespace skl {

// A vector of V elements of T that may sit at any multiple of sizeof(T): rows of odd widths start
// there, and global memory takes a dwordx4 at any address.
template <typename T, int V> struct Unaligned {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};

// Elements [i, i + V) of p as floats; those from `end` on read as `fill` and are not touched.
template <typename T, int V>
__device__ __forceinline__ void load_row(const void *p, uint32_t i, uint32_t end, float (&v)[V], float fill = 0.0f) {
    const T *q = reinterpret_cast<const T *>(p) + i;
    if (i + V <= end) {
        const auto w = *reinterpret_cast<const typename Unaligned<T, V>::type *>(q);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (float)w[e];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = i + e < end ? (float)q[e] : fill;
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_row(void *p, uint32_t i, uint32_t end, const float (&v)[V]) {
    T *q = reinterpret_cast<T *>(p) + i;
    if (i + V <= end) {
        typename Unaligned<T, V>::type w;
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = (T)v[e];
        *reinterpret_cast<typename Unaligned<T, V>::type *>(q) = w;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (i + e < end) q[e] = (T)v[e];
    }
}

__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
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

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

// Elements [i, i + V) of p as floats; those from `end` on read as 0 and are not touched.
template <typename T, int V>
__device__ __forceinline__ void load_row(const void *p, uint32_t i, uint32_t end, float (&v)[V]) {
    const T *q = reinterpret_cast<const T *>(p);
    if (i + V <= end) {
        const auto w = *reinterpret_cast<const typename Unaligned<T, V>::type *>(q + i);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (float)w[e];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = i + e < end ? (float)q[i + e] : 0.0f;
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

// Which of a workgroup's rows a thread has a part in, with NT threads to a row: known to be the
// same in a whole wave where it is, so that the row's addresses stay in scalar registers.
template <int NT> __device__ __forceinline__ uint32_t sub_row() {
    if constexpr (NT >= 256) return 0;
    if constexpr (NT >= 64) return (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / NT));
    return threadIdx.x / NT;
}

// The row `step` behind `row`, or `rows` where there is none: row + step may be past 32 bits.
__device__ __forceinline__ uint32_t next_row(uint32_t row, uint32_t step, uint32_t rows) {
    return row + min(step, rows - row);
}

// A row of `cols` elements over NT threads: thread t has the vectors of 4 at columns 4 (t + NT c) and,
// of the up to three columns behind the last whole vector, the t-th, as its element E.
template <typename T, int E> struct RowPart {
    typename Unaligned<T, 4>::type v[E / 4];
    T last;
};
template <int NT> struct RowMap {
    uint32_t tid, cols;
    __device__ __forceinline__ uint32_t col(int c) const { return (c * NT + tid) * 4; }
    __device__ __forceinline__ uint32_t tail() const { return (cols & ~3u) + tid; }
    __device__ __forceinline__ bool whole(int c) const { return col(c) + 4 <= cols; }
    __device__ __forceinline__ bool tailed() const { return tid < (cols & 3u); }

    // Elements past the row's end are 0.
    template <typename T, int E> __device__ __forceinline__ void read(const void *row, RowPart<T, E> &to) const {
        const T *p = reinterpret_cast<const T *>(row);
        typedef typename Unaligned<T, 4>::type Vec;
#pragma unroll
        for (int c = 0; c < E / 4; ++c) {
            to.v[c] = Vec{};
            if (whole(c)) to.v[c] = *reinterpret_cast<const Vec *>(p + col(c));
        }
        to.last = tailed() ? p[tail()] : (T)0;
    }
    template <typename T, int E> __device__ __forceinline__ void read(const void *row, float (&to)[E + 1]) const {
        RowPart<T, E> part;
        read<T, E>(row, part);
        floats<T, E>(part, to);
    }
    template <typename T, int E> __device__ __forceinline__ static void floats(const RowPart<T, E> &part, float (&to)[E + 1]) {
#pragma unroll
        for (int e = 0; e < E; ++e) to[e] = (float)part.v[e / 4][e % 4];
        to[E] = (float)part.last;
    }
    template <typename T, int E> __device__ __forceinline__ void write(void *row, const float (&from)[E + 1]) const {
        T *p = reinterpret_cast<T *>(row);
        typedef typename Unaligned<T, 4>::type Vec;
#pragma unroll
        for (int c = 0; c < E / 4; ++c) {
            Vec w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = (T)from[4 * c + e];
            if (whole(c)) *reinterpret_cast<Vec *>(p + col(c)) = w;
        }
        if (tailed()) p[tail()] = (T)from[E];
    }
};

// The sums of N values over the NT threads of a row (16 or 64: lanes of one wave), in every one of
// them, in a fixed order.  slots: N NT / 64 floats of LDS that no other sum uses until every
// thread has passed another barrier.
template <int NT, int N> __device__ __forceinline__ void row_sums(float (&v)[N], float *slots) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lanes_sum<(NT < 64 ? NT : 64)>(v[i]);
    if constexpr (NT > 64) {
        constexpr int W = NT / 64;
        if ((threadIdx.x & 63u) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) slots[i * W + (threadIdx.x >> 6)] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) v[i] += slots[i * W + w];
        }
    }
}

}  // namespace skl

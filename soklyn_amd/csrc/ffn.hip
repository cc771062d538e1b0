// ffn.hip — element-wise kernels of the gated feed-forward block, the projection into the stream
// and dropout.
//
// All three are streams over flat, contiguous tensors, HBM-bound: vectors of V elements to a
// thread, whatever the row's length (a vector that crosses into the next row draws its dropout for
// both), element by element where a base is not on 16 bytes and for the last n % V.  V is what 16
// bytes of the widest tensor hold, so that neighbouring lanes' accesses meet: fp32 gradients by
// eights beside fp16 tensors, every second 16 bytes to an instruction, ran 15% slower (16384 x
// 4096, fp16: the gradients of a gated block 277 -> 251 us, of a projection 165 -> 137).
#include "ffn.h"
#include "ffn_epi.h"

namespace skl {

constexpr uint32_t kFlatThreads = 256;
// Workgroups for `items` vectors, `each` of them to a thread past eight workgroups to a CU.  Threads of
// one vector leave the order of the stream to the dispatcher; 2048 workgroups that loop drift apart
// (the gradients of a gated block above: 251 -> 225 us, 6.0 TB/s).  Where a thread starts with a division
// for its row (draws of dropout), two vectors pay for it (projection, 32768 x 256 vectors of 4, fp16 with
// SiLU and dropout: one 67.8 us, two 65.5, 16 68.3; dropout, fp16 4096 x 4096: 15.7, 13.8).
static uint32_t flat_groups(uint64_t items, uint32_t each) {
    const uint64_t all = (items + kFlatThreads - 1) / kFlatThreads, g = (all + each - 1) / each;
    const uint64_t least = all < 2048 ? (all ? all : 1) : 2048, most = 1u << 22;   // (a launch has below 2^32 threads)
    return (uint32_t)(g < least ? least : g < most ? g : most);
}
static bool on16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T, int V> struct FlatVec { T v[V]; };
// 8 or 16 bytes
template <typename T, int V> using FlatBits = uint32_t __attribute__((ext_vector_type(V * sizeof(T) / 4)));
template <typename T, int V> __device__ __forceinline__ void flat_load(const T *p, uint64_t i, float (&to)[V]) {
    if constexpr (V == 1) {
        to[0] = to_f32(p[i]);
    } else {
        const FlatVec<T, V> v =
            __builtin_bit_cast(FlatVec<T, V>, __builtin_nontemporal_load(reinterpret_cast<const FlatBits<T, V> *>(p + i)));
#pragma unroll
        for (int j = 0; j < V; ++j) to[j] = to_f32(v.v[j]);
    }
}
template <typename T, int V> __device__ __forceinline__ void flat_store(T *p, uint64_t i, const float (&from)[V]) {
    if constexpr (V == 1) {
        p[i] = from_f32<T>(from[0]);
    } else {
        FlatVec<T, V> v;
#pragma unroll
        for (int j = 0; j < V; ++j) v.v[j] = from_f32<T>(from[j]);
        __builtin_nontemporal_store(__builtin_bit_cast(FlatBits<T, V>, v), reinterpret_cast<FlatBits<T, V> *>(p + i));
    }
}

// Row and column of a flat index that advances by a fixed step: one division to start with.
struct Place {
    uint32_t row, col, drow, dcol, cols;
    __device__ __forceinline__ Place(uint64_t i, uint64_t step, uint32_t cols_) : cols(cols_) {
        row = (uint32_t)(i / cols);
        col = (uint32_t)(i % cols);
        drow = (uint32_t)(step / cols);
        dcol = (uint32_t)(step % cols);
    }
    __device__ __forceinline__ void next() {
        row += drow;
        const uint64_t c = (uint64_t)col + dcol;
        row += c >= cols;
        col = (uint32_t)(c >= cols ? c - cols : c);
    }
};
// The dropout factors of V consecutive elements from a place on.
template <int V> __device__ __forceinline__ void drop_factors(const DropArgs &d, const Place &at, float (&f)[V]) {
    uint32_t row = at.row, col = at.col, mul = at.col * kDropColMul, key = drop_rowkey(d, row);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        f[j] = drop_factor(d, mul, key);
        mul += kDropColMul;
        if (++col == at.cols) {
            col = 0;
            mul = 0;
            key = drop_rowkey(d, ++row);
        }
    }
}

template <typename T, int V> __device__ __forceinline__ void ungate_at(const UngateArgs &a, uint64_t i) {
    float s[V], g[V], u[V], dg[V], du[V];
    flat_load<float, V>(a.s, i, s);
    flat_load<T, V>(reinterpret_cast<const T *>(a.e.a), i, g);
    flat_load<T, V>(reinterpret_cast<const T *>(a.e.u), i, u);
    float v[V], d[V];
    ffn_act_slope<T>(a.e.act, g, a.e.leaky, v, d);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        dg[j] = settled(s[j] * u[j] * d[j]);
        du[j] = settled(s[j] * v[j]);
    }
    flat_store<float, V>(a.e.d_gate, i, dg);
    flat_store<float, V>(a.e.d_up, i, du);
    if constexpr (sizeof(T) == 2) {
        flat_store<half_t, V>(a.e.d_gate_h, i, dg);
        flat_store<half_t, V>(a.e.d_up_h, i, du);
    }
}
template <typename T, int V> __global__ void __launch_bounds__(kFlatThreads) ungate_kernel(UngateArgs a) {
    const uint64_t id = (uint64_t)blockIdx.x * kFlatThreads + threadIdx.x, step = (uint64_t)gridDim.x * kFlatThreads;
    for (uint64_t i = id * V; i + V <= a.n; i += step * V) ungate_at<T, V>(a, i);
    if (V > 1 && id < a.n % V) ungate_at<T, 1>(a, a.n / V * V + id);
}

template <typename T, int V> __device__ __forceinline__ void unproject_at(const UnprojectArgs &a, uint64_t i, const Place &at) {
    float dh[V], d[V];
    flat_load<float, V>(a.dh, i, dh);
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = dh[j];
    if (a.act) {
        float z[V];
        flat_load<T, V>(reinterpret_cast<const T *>(a.preact), i, z);
        float v[V], slope[V];
        ffn_act_slope<T>(a.act, z, a.leaky, v, slope);
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] *= slope[j];
    }
    if (a.drop.on) {
        float f[V];
        drop_factors<V>(a.drop, at, f);
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = f[j] != 0.0f ? d[j] * f[j] : 0.0f;   // nothing passes a dropped element
    }
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = settled(d[j]);
    flat_store<float, V>(a.d_prenorm, i, d);
    if constexpr (sizeof(T) == 2) flat_store<half_t, V>(a.d_prenorm_h, i, d);
    if (a.dx) {
#pragma unroll
        for (int j = 0; j < V; ++j) dh[j] *= a.scale;
        flat_store<float, V>(a.dx, i, dh);
    }
}
template <typename T, int V> __global__ void __launch_bounds__(kFlatThreads) unproject_kernel(UnprojectArgs a) {
    const uint64_t id = (uint64_t)blockIdx.x * kFlatThreads + threadIdx.x, step = (uint64_t)gridDim.x * kFlatThreads;
    const uint64_t n = (uint64_t)a.rows * a.cols;
    Place at(id * V, step * V, a.cols);
    for (uint64_t i = id * V; i + V <= n; i += step * V, at.next()) unproject_at<T, V>(a, i, at);
    if (V > 1 && id < n % V) {
        const uint64_t i = n / V * V + id;
        unproject_at<T, 1>(a, i, Place(i, 0, a.cols));
    }
}

template <typename T, int V> __device__ __forceinline__ void dropout_at(const DropoutArgs &a, uint64_t i, const Place &at) {
    float x[V], f[V];
    flat_load<T, V>(reinterpret_cast<const T *>(a.in), i, x);
    if (a.drop.on) {
        drop_factors<V>(a.drop, at, f);
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = f[j] != 0.0f ? x[j] * f[j] : 0.0f;
    }
    flat_store<T, V>(reinterpret_cast<T *>(a.out), i, x);
}
template <typename T, int V> __global__ void __launch_bounds__(kFlatThreads) dropout_kernel(DropoutArgs a) {
    const uint64_t id = (uint64_t)blockIdx.x * kFlatThreads + threadIdx.x, step = (uint64_t)gridDim.x * kFlatThreads;
    const uint64_t n = (uint64_t)a.rows * a.cols;
    Place at(id * V, step * V, a.cols);
    for (uint64_t i = id * V; i + V <= n; i += step * V, at.next()) dropout_at<T, V>(a, i, at);
    if (V > 1 && id < n % V) {
        const uint64_t i = n / V * V + id;
        dropout_at<T, 1>(a, i, Place(i, 0, a.cols));
    }
}

template <typename T> static hipError_t ungate_t(const UngateArgs &a, hipStream_t s) {
    constexpr int V = 4;
    const bool vec = on16(a.s) && on16(a.e.a) && on16(a.e.u) && on16(a.e.d_gate) && on16(a.e.d_up) && on16(a.e.d_gate_h) &&
                     on16(a.e.d_up_h);
    if (vec)
        ungate_kernel<T, V><<<flat_groups((a.n + V - 1) / V, 1), kFlatThreads, 0, s>>>(a);
    else
        ungate_kernel<T, 1><<<flat_groups(a.n, 1), kFlatThreads, 0, s>>>(a);
    return hipGetLastError();
}
hipError_t launch_ungate(const UngateArgs &a, uint32_t dtype, hipStream_t s) {
    if (a.n == 0) return hipSuccess;
    return dtype == 1 ? ungate_t<half_t>(a, s) : ungate_t<float>(a, s);
}

template <typename T> static hipError_t unproject_t(const UnprojectArgs &a, hipStream_t s) {
    constexpr int V = 4;
    const uint64_t n = (uint64_t)a.rows * a.cols;
    if (on16(a.dh) && on16(a.preact) && on16(a.d_prenorm) && on16(a.dx) && on16(a.d_prenorm_h))
        unproject_kernel<T, V><<<flat_groups((n + V - 1) / V, 2), kFlatThreads, 0, s>>>(a);
    else
        unproject_kernel<T, 1><<<flat_groups(n, 2), kFlatThreads, 0, s>>>(a);
    return hipGetLastError();
}
hipError_t launch_unproject(const UnprojectArgs &a, uint32_t dtype, hipStream_t s) {
    if (!a.rows || !a.cols) return hipSuccess;
    return dtype == 1 ? unproject_t<half_t>(a, s) : unproject_t<float>(a, s);
}

template <typename T> static hipError_t dropout_t(const DropoutArgs &a, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const uint64_t n = (uint64_t)a.rows * a.cols;
    if (on16(a.in) && on16(a.out))
        dropout_kernel<T, V><<<flat_groups((n + V - 1) / V, 2), kFlatThreads, 0, s>>>(a);
    else
        dropout_kernel<T, 1><<<flat_groups(n, 2), kFlatThreads, 0, s>>>(a);
    return hipGetLastError();
}
hipError_t launch_dropout(const DropoutArgs &a, uint32_t dtype, hipStream_t s) {
    if (!a.rows || !a.cols) return hipSuccess;
    return dtype == 1 ? dropout_t<half_t>(a, s) : dropout_t<float>(a, s);
}

}  // namespace skl

// ffn_epi.h — epilogues of the products in ffn.h, in the forms that gemm_dma.h and gemm_wave.h call.
//
// All of them compute from the fp32 sums: the activation reads z before it is rounded into its
// cache (a result kept in 32 bits would otherwise carry the cache's 2^-12), so an output is rounded
// once, where it is stored.
#pragma once

#include <type_traits>

#include "epilogue.h"
#include "ffn.h"

namespace skl {

// Activations of these operators, for both types from the hardware's exp2 and reciprocal but for
// fp32 blocks' Mish; tanh by its series near 0 (tanhf is several times the work of the rest).  Mish is z
// and its slope 1 above 20, where tanh(softplus(z)) is off 1 by 2 e^-40 at most: the blocks' forms say
// NaN from 88.7 on, where e^z overflows, as the reference does; these operators have none to follow.
// N at a time: the choice of the activation outside the elements, whose chains of exp and reciprocal
// then run beside each other.
template <typename T, uint32_t ACT, bool SLOPE, int N>
__device__ __forceinline__ void ffn_act_as(const float (&z)[N], float leaky, float (&v)[N], float (&d)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const bool far = ACT == 7 && z[j] > 20.0f;
        v[j] = ACT == 4 ? tanh_fast(z[j]) : far ? z[j] : activation<T>(ACT, z[j], leaky);
        if constexpr (SLOPE) d[j] = far ? 1.0f : activation_derivative<T>(ACT, 1.0f, v[j], z[j], leaky);
    }
}
template <typename T, bool SLOPE, int N>
__device__ __forceinline__ void ffn_act_n(uint32_t act, const float (&z)[N], float leaky, float (&v)[N], float (&d)[N]) {
    switch (act) {
    case 1: return ffn_act_as<T, 1, SLOPE>(z, leaky, v, d);
    case 2: return ffn_act_as<T, 2, SLOPE>(z, leaky, v, d);
    case 3: return ffn_act_as<T, 3, SLOPE>(z, leaky, v, d);
    case 4: return ffn_act_as<T, 4, SLOPE>(z, leaky, v, d);
    case 6: return ffn_act_as<T, 6, SLOPE>(z, leaky, v, d);
    case 7: return ffn_act_as<T, 7, SLOPE>(z, leaky, v, d);
    default: return ffn_act_as<T, 0, SLOPE>(z, leaky, v, d);
    }
}
// The activations of z in place, or its activations and slopes.
template <typename T, int N> __device__ __forceinline__ void ffn_act(uint32_t act, float (&z)[N], float leaky) {
    float v[N];
    ffn_act_n<T, false>(act, z, leaky, v, v);
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = v[j];
}
template <typename T, int N>
__device__ __forceinline__ void ffn_act_slope(uint32_t act, const float (&z)[N], float leaky, float (&v)[N], float (&d)[N]) {
    ffn_act_n<T, true>(act, z, leaky, v, d);
}

// A gradient as it is stored in fp32: without this its fp16 copy may be made from the product in front
// of that rounding (one mixed-precision multiply), a step away from f16(gradient) now and then.
__device__ __forceinline__ float settled(float v) {
    asm("" : "+v"(v));
    return v;
}

template <typename V> struct Vec4 { typedef f32x4 type; };
template <> struct Vec4<half_t> { typedef f16x4 type; };
template <typename T> __device__ __forceinline__ typename Vec4<T>::type load_nt(const void *p, uint64_t i) {
    return __builtin_nontemporal_load(reinterpret_cast<const typename Vec4<T>::type *>(reinterpret_cast<const T *>(p) + i));
}
__device__ __forceinline__ void st8h_nt(void *p, uint64_t idx, f32x4 lo, f32x4 hi) {
    const half_t h[8] = {(half_t)lo[0], (half_t)lo[1], (half_t)lo[2], (half_t)lo[3],
                         (half_t)hi[0], (half_t)hi[1], (half_t)hi[2], (half_t)hi[3]};
    __builtin_nontemporal_store(*reinterpret_cast<const u32x4 *>(h),
                                reinterpret_cast<u32x4 *>(reinterpret_cast<half_t *>(p) + idx));
}

// ---- both projections of a gated block ---------------------------------------------------
template <typename T> struct EpiPairK {
    typedef PairEpi Params;
    static constexpr bool kPair = true;
    struct Pre {};   // nothing is read per element
    struct Col { f32x4 g, u; };
    struct Col1 { float g, u; };
    struct Col8 { f32x4 g0, g1, u0, u1; };
    __device__ __forceinline__ static uint32_t ldc(const PairEpi &e) { return e.ldc; }
    __device__ __forceinline__ static f32x4 bias4(const void *b, uint32_t n) {
        return b ? load4<T>(b, n) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __device__ __forceinline__ static Col column(const PairEpi &e, uint32_t n) {
        return Col{bias4(e.bias, n), bias4(e.bias2, n)};
    }
    __device__ __forceinline__ static Col1 column1(const PairEpi &e, uint32_t n) {
        return Col1{e.bias ? to_f32(ld_t<T>(e.bias, n)) : 0.0f, e.bias2 ? to_f32(ld_t<T>(e.bias2, n)) : 0.0f};
    }
    __device__ __forceinline__ static Col8 column8(const PairEpi &e, uint32_t n) {
        return Col8{bias4(e.bias, n), bias4(e.bias, n + 4), bias4(e.bias2, n), bias4(e.bias2, n + 4)};
    }
    __device__ __forceinline__ static void finish(const PairEpi &e, uint64_t idx, floatx4 g, floatx4 u, const Col &c) {
        const f32x4 a = g + c.g, v = u + c.u;
        float o[4] = {a[0], a[1], a[2], a[3]};
        ffn_act<T>(e.act, o, e.leaky);
        store4_nt<T>(e.out, idx, f32x4{o[0] * v[0], o[1] * v[1], o[2] * v[2], o[3] * v[3]});
        if (e.a) store4_nt<T>(e.a, idx, a);
        if (e.u) store4_nt<T>(e.u, idx, v);
    }
    // 8 columns (fp16): 16-byte stores
    __device__ __forceinline__ static void finish8(const PairEpi &e, uint64_t idx, floatx4 g0, floatx4 g1, floatx4 u0,
                                                   floatx4 u1, const Col8 &c) {
        const f32x4 a0 = g0 + c.g0, a1 = g1 + c.g1, v0 = u0 + c.u0, v1 = u1 + c.u1;
        float o[8] = {a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
        ffn_act<T>(e.act, o, e.leaky);
        st8h_nt(e.out, idx, f32x4{o[0] * v0[0], o[1] * v0[1], o[2] * v0[2], o[3] * v0[3]},
                f32x4{o[4] * v1[0], o[5] * v1[1], o[6] * v1[2], o[7] * v1[3]});
        if (e.a) st8h_nt(e.a, idx, a0, a1);
        if (e.u) st8h_nt(e.u, idx, v0, v1);
    }
    __device__ __forceinline__ static void apply1(const PairEpi &e, uint32_t m, uint32_t n, float g, float u, const Col1 &c) {
        const uint64_t idx = (uint64_t)m * e.ldc + n;
        const float a = g + c.g, v = u + c.u;
        float o[1] = {a};
        ffn_act<T>(e.act, o, e.leaky);
        st_t<T>(e.out, idx, from_f32<T>(o[0] * v));
        if (e.a) st_t<T>(e.a, idx, from_f32<T>(a));
        if (e.u) st_t<T>(e.u, idx, from_f32<T>(v));
    }
};

// ---- the gradients of a gated block's projections ------------------------------------------
// dg = s * u * act'(a), du = s * act(a)
template <typename T> struct EpiUngateK {
    typedef UngateEpi Params;
    typedef typename Vec4<T>::type V4;
    static constexpr bool kReads = true;
    struct Pre { V4 a, u; };
    struct Pre1 { T a, u; };
    struct Col {};
    struct Col1 {};
    __device__ __forceinline__ static uint32_t ldc(const UngateEpi &e) { return e.ldc; }
    __device__ __forceinline__ static UngateEpi at_split(const UngateEpi &e, uint32_t) { return e; }
    __device__ __forceinline__ static Col column(const UngateEpi &, uint32_t) { return Col{}; }
    __device__ __forceinline__ static Col1 column1(const UngateEpi &, uint32_t) { return Col1{}; }
    __device__ __forceinline__ static void load(const UngateEpi &e, uint64_t idx, uint32_t, Pre &q) {
        q.a = load_nt<T>(e.a, idx);   // read once
        q.u = load_nt<T>(e.u, idx);
    }
    __device__ __forceinline__ static void finish(const UngateEpi &e, uint64_t idx, uint32_t, uint32_t, floatx4 s, const Col &,
                                                  const Pre &q) {
        const float a[4] = {(float)q.a[0], (float)q.a[1], (float)q.a[2], (float)q.a[3]};
        float v[4], d[4];
        ffn_act_slope<T>(e.act, a, e.leaky, v, d);
        f32x4 dg, du;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            dg[j] = settled(s[j] * (float)q.u[j] * d[j]);
            du[j] = settled(s[j] * v[j]);
        }
        __builtin_nontemporal_store(dg, reinterpret_cast<f32x4 *>(e.d_gate + idx));
        __builtin_nontemporal_store(du, reinterpret_cast<f32x4 *>(e.d_up + idx));
        if constexpr (sizeof(T) == 2) {
            store4_nt<half_t>(e.d_gate_h, idx, dg);   // (past the caches: 16384 x 4096, K 2048: 421 -> 395 us)
            store4_nt<half_t>(e.d_up_h, idx, du);
        }
    }
    __device__ __forceinline__ static void load1(const UngateEpi &e, uint64_t idx, Pre1 &q) {
        q.a = ld_t<T>(e.a, idx);
        q.u = ld_t<T>(e.u, idx);
    }
    __device__ __forceinline__ static void finish1(const UngateEpi &e, uint64_t idx, uint32_t, uint32_t, float s, const Col1 &,
                                                   const Pre1 &q) {
        const float a[1] = {to_f32(q.a)};
        float v[1], d[1];
        ffn_act_slope<T>(e.act, a, e.leaky, v, d);
        const float dg = settled(s * to_f32(q.u) * d[0]), du = settled(s * v[0]);
        e.d_gate[idx] = dg;
        e.d_up[idx] = du;
        if constexpr (sizeof(T) == 2) {
            e.d_gate_h[idx] = (half_t)dg;
            e.d_up_h[idx] = (half_t)du;
        }
    }
    __device__ __forceinline__ static void apply1(const UngateEpi &e, uint32_t m, uint32_t n, float s, const Col1 &c, uint32_t) {
        const uint64_t idx = (uint64_t)m * e.ldc + n;
        Pre1 q;
        load1(e, idx, q);
        finish1(e, idx, m, n, s, c, q);
    }
};

// ---- the projection into the stream ---------------------------------------------------------
template <typename T, typename R> struct EpiProjectK {
    typedef ProjectEpi Params;
    typedef typename Vec4<R>::type V4;
    static constexpr bool kReads = true;
    struct Pre { V4 x; };
    struct Pre1 { R x; };
    struct Col { f32x4 bias; };
    struct Col1 { float bias; };
    __device__ __forceinline__ static uint32_t ldc(const ProjectEpi &e) { return e.ldc; }
    __device__ __forceinline__ static ProjectEpi at_split(const ProjectEpi &e, uint32_t) { return e; }
    __device__ __forceinline__ static Col column(const ProjectEpi &e, uint32_t n) {
        return Col{e.bias ? load4<T>(e.bias, n) : f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
    }
    __device__ __forceinline__ static Col1 column1(const ProjectEpi &e, uint32_t n) {
        return Col1{e.bias ? to_f32(ld_t<T>(e.bias, n)) : 0.0f};
    }
    __device__ __forceinline__ static void load(const ProjectEpi &e, uint64_t idx, uint32_t, Pre &q) {
        q.x = e.x ? load_nt<R>(e.x, idx) : V4{0, 0, 0, 0};
    }
    // a dropped element is 0 whatever its value (an infinity too)
    __device__ __forceinline__ static float dropped(const ProjectEpi &e, float v, uint32_t colmul, uint32_t rowkey) {
        return dropout_bits(colmul, rowkey) >= e.drop.keep_min ? v * e.drop.scale : 0.0f;
    }
    __device__ __forceinline__ static void finish(const ProjectEpi &e, uint64_t idx, uint32_t m, uint32_t n, floatx4 s,
                                                  const Col &c, const Pre &q) {
        const f32x4 z = s + c.bias;
        if (e.preact) store4_nt<T>(e.preact, idx, z);
        float a[4] = {z[0], z[1], z[2], z[3]};
        ffn_act<T>(e.act, a, e.leaky);
        f32x4 v = {a[0], a[1], a[2], a[3]};
        if (e.drop.on) {
            const uint32_t rk = drop_rowkey(e.drop, m);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = dropped(e, v[j], (n + j) * kDropColMul, rk);
        }
        if (e.x) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = fmaf(e.scale, (float)q.x[j], v[j]);
        }
        store4_nt<R>(e.h, idx, v);
    }
    __device__ __forceinline__ static void load1(const ProjectEpi &e, uint64_t idx, Pre1 &q) {
        q.x = e.x ? ld_t<R>(e.x, idx) : (R)0;
    }
    __device__ __forceinline__ static void finish1(const ProjectEpi &e, uint64_t idx, uint32_t m, uint32_t n, float s,
                                                   const Col1 &c, const Pre1 &q) {
        const float z = s + c.bias;
        if (e.preact) st_t<T>(e.preact, idx, from_f32<T>(z));
        float a[1] = {z};
        ffn_act<T>(e.act, a, e.leaky);
        float v = a[0];
        if (e.drop.on) v = dropped(e, v, n * kDropColMul, drop_rowkey(e.drop, m));
        if (e.x) v = fmaf(e.scale, to_f32(q.x), v);
        st_t<R>(e.h, idx, from_f32<R>(v));
    }
    __device__ __forceinline__ static void apply1(const ProjectEpi &e, uint32_t m, uint32_t n, float s, const Col1 &c, uint32_t) {
        const uint64_t idx = (uint64_t)m * e.ldc + n;
        Pre1 q;
        load1(e, idx, q);
        finish1(e, idx, m, n, s, c, q);
    }
};

// ---- the sum of two products, stored in fp32 -------------------------------------------------
struct EpiChainK {
    typedef ChainEpi Params;
    static constexpr bool kChain = true;
    static constexpr int kDmaSpacing = 1;     // as EpiStoreK
    static constexpr int kReadsPerMfma = 1;
    static constexpr bool kDirect = true;
    static constexpr int kDirectBatch = 8;
    struct Pre {};
    struct Col {};
    struct Col1 {};
    __device__ __forceinline__ static uint32_t ldc(const ChainEpi &e) { return e.ldc; }
    __device__ __forceinline__ static ChainEpi at_split(const ChainEpi &e, uint32_t) { return e; }
    __device__ __forceinline__ static Col column(const ChainEpi &, uint32_t) { return Col{}; }
    __device__ __forceinline__ static Col1 column1(const ChainEpi &, uint32_t) { return Col1{}; }
    __device__ __forceinline__ static void load(const ChainEpi &, uint64_t, uint32_t, Pre &) {}
    __device__ __forceinline__ static void finish(const ChainEpi &e, uint64_t idx, uint32_t, uint32_t, floatx4 v, const Col &,
                                                  const Pre &) {
        __builtin_nontemporal_store(v, reinterpret_cast<floatx4 *>(e.out + idx));
    }
    __device__ __forceinline__ static void direct(const ChainEpi &e, uint64_t idx, uint32_t, uint32_t, floatx4 v, const Pre &) {
        *reinterpret_cast<floatx4 *>(e.out + idx) = v;
    }
    __device__ __forceinline__ static void apply1(const ChainEpi &e, uint32_t m, uint32_t n, float v, const Col1 &, uint32_t) {
        e.out[(uint64_t)m * e.ldc + n] = v;
    }
    __device__ __forceinline__ static void apply(const ChainEpi &e, const GemmShape &sh, uint32_t m, uint32_t n, floatx4 v,
                                                 uint32_t) {
        if (m >= sh.M) return;
        float *o = e.out + (uint64_t)m * e.ldc + n;
        if (n + 3 < sh.N) {
            *reinterpret_cast<floatx4 *>(o) = v;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < sh.N) o[j] = v[j];
        }
    }
};

}  // namespace skl

// mxfp4.hip — matrices to 4-bit microscaled floats and back, and the product of two.
#include "mx_gemm.h"
#include "mxfp4.h"
#include "rows.h"

namespace skl {

namespace {

// The scale byte of a block from its largest magnitude: 2^(e - 2) with 2^e the largest power of
// two up to it, so that it lies in [4, 8) of the scale (6 is the largest code; past it values
// saturate).  255 where the block holds an infinity or NaN.  bits: of the magnitude as fp32.
__device__ __forceinline__ uint32_t mx_scale(uint32_t bits) {
    const uint32_t e = bits >> 23;
    return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}

// Eight values of one block to codes, the first in the lowest half byte.  The convert rounds to
// nearest, ties to the even code, and saturates.  It takes its scale as a power of two in fp32,
// which for the smallest (byte 0: 2^-127) would be subnormal: 2^64 goes to the values instead.
__device__ __forceinline__ uint32_t mx_codes(const float (&v)[8], uint32_t scale) {
    const bool low = scale < 64u;
    const float up = low ? 0x1p64f : 1.0f;
    const float s = __builtin_bit_cast(float, (scale == 255u ? 254u : low ? scale + 64u : scale) << 23);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0] * up, v[1] * up, s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2] * up, v[3] * up, s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4] * up, v[5] * up, s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6] * up, v[7] * up, s, 3);
    return c;
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// The value of a code: its magnitude is exact in fp32, and so is its product with any scale.
__device__ __forceinline__ float mx_value(uint32_t code, uint32_t scale) {
    const uint32_t c = code & 7u;
    // 0, 0.5, then 1.m 2^(e - 1)
    float v = c < 2u ? 0.5f * (float)c : __builtin_bit_cast(float, ((c >> 1) + 126u) << 23 | (c & 1u) << 22);
    v = code & 8u ? -v : v;
    return scale == 255u ? __builtin_nanf("") : ldexpf(v, (int)scale - 127);
}

// Vectors along the rows of a [n x k] matrix: four lanes to a block of 32, eight elements each.
template <typename T> __global__ void __launch_bounds__(256) mx_quantise_kernel(MxCastArgs a) {
    const uint32_t kp = mx_pad(a.k), lanes = kp / 8;   // lanes of a vector
    const uint64_t total = (uint64_t)a.n * lanes;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        const uint32_t row = (uint32_t)(i / lanes), l = (uint32_t)(i % lanes);
        float v[8];
        load_row<T, 8>(reinterpret_cast<const T *>(a.values) + (uint64_t)row * a.k, l * 8, a.k, v);
        uint32_t big = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) big = max(big, magnitude(v[e]));
        big = max(big, (uint32_t)__shfl_xor((int)big, 1, 64));
        big = max(big, (uint32_t)__shfl_xor((int)big, 2, 64));
        const uint32_t scale = mx_scale(big);
        reinterpret_cast<uint32_t *>(a.codes)[i] = mx_codes(v, scale);
        if ((l & 3u) == 0) a.scales[i / 4] = (uint8_t)scale;
    }
}

template <typename T> __global__ void __launch_bounds__(256) mx_dequantise_kernel(MxCastArgs a) {
    const uint32_t lanes = mx_pad(a.k) / 8;
    const uint64_t total = (uint64_t)a.n * lanes;
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (uint64_t)gridDim.x * 256) {
        const uint32_t row = (uint32_t)(i / lanes), l = (uint32_t)(i % lanes);
        const uint32_t c = reinterpret_cast<const uint32_t *>(a.codes)[i], scale = a.scales[i / 4];
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = mx_value(c >> 4 * e, scale);
        if (l * 8 < a.k) store_row<T, 8>(reinterpret_cast<T *>(a.values) + (uint64_t)row * a.k, l * 8, a.k, v);
    }
}

// Vectors down the columns of a [k x n] matrix: a workgroup takes 64 columns by 128 rows, a wave
// one block of 32 rows (a row's 64 elements are one load); the codes go through LDS, so that each
// vector's 64 bytes are written together.
template <typename T> __global__ void __launch_bounds__(256) mx_quantise_down_kernel(MxCastArgs a) {
    __shared__ u32x4 codes[64][5];
    __shared__ uint8_t scales[64][4];
    const uint32_t kp = mx_pad(a.k), ntiles = (a.n + 63u) / 64u;
    const uint32_t ntile = blockIdx.x % ntiles, ktile = blockIdx.x / ntiles;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t k0 = ktile * 128u + wave * 32u, col = ntile * 64u + lane;
    float v[32];
    uint32_t big = 0;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        v[e] = col < a.n && k0 + e < a.k ? (float)reinterpret_cast<const T *>(a.values)[(uint64_t)(k0 + e) * a.n + col] : 0.0f;
        big = max(big, magnitude(v[e]));
    }
    const uint32_t scale = mx_scale(big);
    u32x4 c;
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = mx_codes(*reinterpret_cast<const float (*)[8]>(&v[8 * e]), scale);
    codes[lane][wave] = c;
    scales[lane][wave] = (uint8_t)scale;
    __syncthreads();
    const uint32_t vec = threadIdx.x >> 2, part = threadIdx.x & 3u, to = ntile * 64u + vec;
    if (to < a.n)
        reinterpret_cast<u32x4 *>(a.codes + (uint64_t)to * (kp / 2) + ktile * 64u)[part] = codes[vec][part];
    if (threadIdx.x < 64 && col < a.n)
        *reinterpret_cast<uint32_t *>(a.scales + (uint64_t)col * (kp / 32) + ktile * 4u) =
            *reinterpret_cast<const uint32_t *>(scales[lane]);
}

template <typename T> __global__ void __launch_bounds__(256) mx_dequantise_down_kernel(MxCastArgs a) {
    __shared__ u32x4 codes[64][5];
    const uint32_t kp = mx_pad(a.k), ntiles = (a.n + 63u) / 64u;
    const uint32_t ntile = blockIdx.x % ntiles, ktile = blockIdx.x / ntiles;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t vec = threadIdx.x >> 2, part = threadIdx.x & 3u, from = ntile * 64u + vec;
    if (from < a.n)
        codes[vec][part] = reinterpret_cast<const u32x4 *>(a.codes + (uint64_t)from * (kp / 2) + ktile * 64u)[part];
    __syncthreads();
    const uint32_t k0 = ktile * 128u + wave * 32u, col = ntile * 64u + lane;
    if (col >= a.n) return;
    const uint32_t scale = a.scales[(uint64_t)col * (kp / 32) + k0 / 32u];
    const u32x4 c = codes[lane][wave];
#pragma unroll
    for (int e = 0; e < 32; ++e)
        if (k0 + e < a.k)
            reinterpret_cast<T *>(a.values)[(uint64_t)(k0 + e) * a.n + col] = (T)mx_value(c[e / 8] >> 4 * (e % 8), scale);
}

// A lane's block of 32 elements of x, from element i of a row of k, as the product's operand.
template <typename T>
__device__ __forceinline__ u32x4 mx_block(const T *row, uint32_t i, uint32_t k, uint32_t &scale) {
    float v[4][8];
    uint32_t big = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        load_row<T, 8>(row, i + 8 * c, k, v[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) big = max(big, magnitude(v[c][e]));
    }
    scale = mx_scale(big);
    return u32x4{mx_codes(v[0], scale), mx_codes(v[1], scale), mx_codes(v[2], scale), mx_codes(v[3], scale)};
}

__device__ __forceinline__ void mx_mma_plain(f32x4 &acc, const u32x4 &w, uint32_t ws, const u32x4 &x, uint32_t xs) {
    const intx8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const intx8 b = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, 0, (int)ws, 0, (int)xs);
}

// 16 x 16 outputs of a wave: lane holds columns col .. + 3 of a row.
template <typename T>
__device__ __forceinline__ void mx_store(const MxForwardArgs &a, f32x4 s, uint32_t row, uint32_t col) {
    if (row >= a.m || col >= a.n) return;
    float v[4], b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (a.bias) load_row<T, 4>(a.bias, col, a.n, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = s[e] + b[e];
    activate(a.act, a.leaky, v);
    store_row<T, 4>(reinterpret_cast<T *>(a.out) + (uint64_t)row * a.n, col, a.n, v);
}

// Few rows: x in 4 bits times w in one launch, tiles of 16 MT rows by 16 columns.  The operand of
// v_mfma_scale_16x16x128 is one block of 32 consecutive elements of one vector per lane (vector
// lane % 16, block lane / 16) with that block's scale, so w goes from memory to the matrix cores
// as it is stored, and a lane turns 32 elements of x into its operand by itself.  The eight waves
// of a workgroup take every eighth step of 128 of the k axis, with the loads of U steps in flight,
// and their sums are joined in LDS in the order of the waves.
template <typename T, int MT, int U> __global__ void __launch_bounds__(512) mx_rows_kernel(MxForwardArgs a) {
    constexpr int WV = 8;
    typedef typename Unaligned<T, 8>::type Vec;
    __shared__ f32x4 part[WV][MT][64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, r = lane & 15u, g = lane >> 4;
    const uint32_t n0 = blockIdx.x * 16u;
    const uint32_t kp = mx_pad(a.k);
    // rows past an operand's end read its last one; what they give is not stored
    const uint32_t wn = min(n0 + r, a.n - 1);
    const uint8_t *wc = a.w_codes + (uint64_t)wn * (kp / 2), *wsc = a.w_scales + (uint64_t)wn * (kp / 32);
    const T *x[MT];
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        x[i] = reinterpret_cast<const T *>(a.x) + (uint64_t)min(16u * i + r, a.m - 1) * a.k;
        acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (uint32_t k0 = wave * 128u; k0 < kp; k0 += U * WV * 128u) {
        u32x4 w[U];
        uint32_t ws[U];
        Vec v[U][MT][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t k = k0 + u * WV * 128u + g * 32u;
            if (k >= kp) break;
            w[u] = *reinterpret_cast<const u32x4 *>(wc + k / 2);
            ws[u] = wsc[k / 32];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint32_t e0 = k + 8 * c;
                    v[u][i][c] = Vec{};
                    if (e0 + 8 <= a.k)
                        v[u][i][c] = *reinterpret_cast<const Vec *>(x[i] + e0);
                    else
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (e0 + e < a.k) v[u][i][c][e] = x[i][e0 + e];
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k0 + u * WV * 128u >= kp) break;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                uint32_t big = 0;
                float f[4][8];
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        f[c][e] = (float)v[u][i][c][e];
                        big = max(big, magnitude(f[c][e]));
                    }
                const uint32_t xs = mx_scale(big);
                const u32x4 xc = {mx_codes(f[0], xs), mx_codes(f[1], xs), mx_codes(f[2], xs), mx_codes(f[3], xs)};
                mx_mma_plain(acc[i], w[u], ws[u], xc, xs);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave >= MT) return;
    f32x4 s = part[0][wave][lane];
#pragma unroll
    for (int w = 1; w < WV; ++w) s += part[w][wave][lane];
    mx_store<T>(a, s, 16u * wave + r, n0 + 4u * g);
}

// Ordinary batches: 64 x 64 tiles over staged codes and scales (below), whose waves split the k axis
// as above, fragments straight from memory to registers.
template <typename T> __global__ void __launch_bounds__(512) mx_split_kernel(MxForwardArgs a, MxGemmArgs t) {
    constexpr int WV = 8;
    __shared__ f32x4 part[WV][16][64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, r = lane & 15u, g = lane >> 4;
    uint32_t tm, tn;
    tile_coords(blockIdx.x, t.tiles_m, t.tiles_n, tm, tn);
    const uint32_t m0 = tm * 64u, n0 = tn * 64u, xp = t.k2 / 2, wp = t.kp / 2;
    const uint8_t *x = t.x + (uint64_t)(m0 + r) * xp + g * 16u, *w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = t.w + (uint64_t)min(n0 + 16u * j + r, a.n - 1) * wp + g * 16u;
    const uint32_t *xs = reinterpret_cast<const uint32_t *>(t.xs) + ((uint64_t)tm * (t.k2 / 32) + g) * 16u + r;
    const uint32_t *ws = reinterpret_cast<const uint32_t *>(t.ws) + ((uint64_t)tn * (t.k2 / 32) + g) * 16u + r;
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i / 4][i % 4] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 2
    for (uint32_t step = wave; step < t.kp / 128u; step += WV) {
        u32x4 fx[4], fw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) fx[i] = *reinterpret_cast<const u32x4 *>(x + 16u * i * xp + step * 64u);
#pragma unroll
        for (int j = 0; j < 4; ++j) fw[j] = *reinterpret_cast<const u32x4 *>(w[j] + step * 64u);
        const uint32_t sx = xs[step * 64u], sw = ws[step * 64u];
        Each<16>::run([&](auto q) {
            constexpr int I = decltype(q)::value / 4, J = decltype(q)::value % 4;
            const intx8 wo = {(int)fw[J][0], (int)fw[J][1], (int)fw[J][2], (int)fw[J][3], 0, 0, 0, 0};
            const intx8 xo = {(int)fx[I][0], (int)fx[I][1], (int)fx[I][2], (int)fx[I][3], 0, 0, 0, 0};
            acc[I][J] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wo, xo, acc[I][J], 4, 4, J, (int)sw, I, (int)sx);
        });
    }
#pragma unroll
    for (int q = 0; q < 16; ++q) part[wave][q][lane] = acc[q / 4][q % 4];
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t q = 2 * wave + h;
        f32x4 s = part[0][q][lane];
#pragma unroll
        for (int v = 1; v < WV; ++v) s += part[v][q][lane];
        mx_store<T>(a, s, m0 + 16u * (q / 4) + r, n0 + 16u * (q % 4) + 4u * g);
    }
}

// What the tiled product reads: x [m x k] as codes [mp x k2 / 2], and both operands' scales in its
// order (mx_gemm.h).  A workgroup takes 64 vectors by 128 elements, a thread one block; the first
// `xtiles` workgroups x, the others w's scales.  Vectors and elements past the matrix are 0.
struct MxStageArgs {
    uint32_t m, n, k, kp, k2, xtiles;
    const void *x;
    const uint8_t *w_scales;
    uint8_t *codes, *xs, *ws;
};
template <typename T> __global__ void __launch_bounds__(256) mx_stage_kernel(MxStageArgs a) {
    __shared__ uint32_t words[4][16];
    const uint32_t ktiles = a.k2 / 128u, vec = threadIdx.x >> 2, block = threadIdx.x & 3u;
    const bool is_w = blockIdx.x >= a.xtiles;
    const uint32_t tile = is_w ? blockIdx.x - a.xtiles : blockIdx.x, group = tile / ktiles, kt = tile % ktiles;
    const uint32_t v = group * 64u + vec, kb = kt * 4u + block;
    uint32_t scale = 0;
    if (is_w) {
        if (v < a.n && kb < a.kp / 32u) scale = a.w_scales[(uint64_t)v * (a.kp / 32u) + kb];
    } else {
        u32x4 c = {0, 0, 0, 0};
        if (v < a.m) c = mx_block(reinterpret_cast<const T *>(a.x) + (uint64_t)v * a.k, kb * 32u, a.k, scale);
        *reinterpret_cast<u32x4 *>(a.codes + (uint64_t)v * (a.k2 / 2u) + kb * 16u) = c;
    }
    reinterpret_cast<uint8_t *>(words)[block * 64u + (vec & 15u) * 4u + (vec >> 4)] = (uint8_t)scale;
    __syncthreads();
    if (threadIdx.x < 64)
        reinterpret_cast<uint32_t *>(is_w ? a.ws : a.xs)[((uint64_t)group * (a.k2 / 32u) + kt * 4u) * 16u + threadIdx.x] =
            words[threadIdx.x >> 4][threadIdx.x & 15u];
}

// BT: the tile edge, 64, 128 or 256.
template <typename T, int BT> hipError_t mx_tiles_t(const MxForwardArgs &f, hipStream_t s) {
    const MxWork w = mx_work(f.k, f.n, f.m);
    MxStageArgs st{};
    MxGemmArgs a{};
    a.m = st.m = f.m;
    a.n = st.n = f.n;
    st.k = f.k;
    a.kp = st.kp = mx_pad(f.k);
    a.k2 = st.k2 = w.k2;
    st.x = f.x;
    st.w_scales = f.w_scales;
    st.codes = reinterpret_cast<uint8_t *>(f.work);
    st.xs = st.codes + w.codes;
    st.ws = st.xs + w.xs;
    a.x = st.codes;
    a.xs = st.xs;
    a.ws = st.ws;
    a.w = f.w_codes;
    a.bias = f.bias;
    a.act = f.act;
    a.leaky = f.leaky;
    a.out = f.out;
    a.tiles_m = (f.m + BT - 1) / BT;
    a.tiles_n = (f.n + BT - 1) / BT;
    st.xtiles = w.mp / 64u * (w.k2 / 128u);
    hipLaunchKernelGGL(mx_stage_kernel<T>, dim3(st.xtiles + w.np / 64u * (w.k2 / 128u)), dim3(256), 0, s, st);
    if constexpr (BT == 64)
        hipLaunchKernelGGL(mx_split_kernel<T>, dim3(a.tiles_m * a.tiles_n), dim3(512), 0, s, f, a);
    else
        hipLaunchKernelGGL((mx_gemm_kernel<T, BT>), dim3(a.tiles_m * a.tiles_n), dim3(2 * BT), 0, s, a);
    return hipGetLastError();
}

template <typename T> hipError_t mx_forward_t(const MxForwardArgs &a, hipStream_t s) {
    switch (mx_tile(a.m, a.n)) {
    case 256: return mx_tiles_t<T, 256>(a, s);
    case 128: return mx_tiles_t<T, 128>(a, s);
    case 64: return mx_tiles_t<T, 64>(a, s);
    default: break;
    }
    // fewer elements in flight where a row's are twice as large or there are twice as many rows
    constexpr int U = sizeof(T) == 2 ? 4 : 2;
    if (a.m <= 16)
        hipLaunchKernelGGL((mx_rows_kernel<T, 1, U>), dim3((a.n + 15) / 16), dim3(512), 0, s, a);
    else
        hipLaunchKernelGGL((mx_rows_kernel<T, 2, U / 2>), dim3((a.n + 15) / 16), dim3(512), 0, s, a);
    return hipGetLastError();
}

dim3 flat_grid(uint64_t items) { return dim3((uint32_t)(items / 256 + 1 < 8192 ? items / 256 + 1 : 8192)); }
dim3 down_grid(const MxCastArgs &a) { return dim3((a.n + 63) / 64 * (mx_pad(a.k) / 128)); }

}  // namespace

hipError_t launch_mx_quantise(const MxCastArgs &a, uint32_t dtype, bool down, hipStream_t s) {
    if (a.n == 0 || a.k == 0) return hipSuccess;
    const uint64_t items = (uint64_t)a.n * (mx_pad(a.k) / 8);
    if (down && dtype)
        hipLaunchKernelGGL(mx_quantise_down_kernel<half_t>, down_grid(a), dim3(256), 0, s, a);
    else if (down)
        hipLaunchKernelGGL(mx_quantise_down_kernel<float>, down_grid(a), dim3(256), 0, s, a);
    else if (dtype)
        hipLaunchKernelGGL(mx_quantise_kernel<half_t>, flat_grid(items), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(mx_quantise_kernel<float>, flat_grid(items), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_mx_dequantise(const MxCastArgs &a, uint32_t dtype, bool down, hipStream_t s) {
    if (a.n == 0 || a.k == 0) return hipSuccess;
    const uint64_t items = (uint64_t)a.n * (mx_pad(a.k) / 8);
    if (down && dtype)
        hipLaunchKernelGGL(mx_dequantise_down_kernel<half_t>, down_grid(a), dim3(256), 0, s, a);
    else if (down)
        hipLaunchKernelGGL(mx_dequantise_down_kernel<float>, down_grid(a), dim3(256), 0, s, a);
    else if (dtype)
        hipLaunchKernelGGL(mx_dequantise_kernel<half_t>, flat_grid(items), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(mx_dequantise_kernel<float>, flat_grid(items), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_mx_forward(const MxForwardArgs &a, uint32_t dtype, hipStream_t s) {
    return dtype ? mx_forward_t<half_t>(a, s) : mx_forward_t<float>(a, s);
}

}  // namespace skl

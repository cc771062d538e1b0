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

// The largest magnitude of the block whose eight elements each of four neighbouring lanes has.
__device__ __forceinline__ uint32_t mx_top4(const float (&v)[8]) {
    uint32_t big = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) big = max(big, magnitude(v[e]));
    big = max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, 0xB1, 0xf, 0xf, true));          // quad_perm 1 0 3 2
    return max(big, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)big, 0x4E, 0xf, 0xf, true));   // quad_perm 2 3 0 1
}

// Eight codes, the first in the lowest half byte, as the values they stand for: the convert's are
// exact, and so is their product with any scale.
__device__ __forceinline__ void mx_values(uint32_t codes, uint32_t scale, float (&v)[8]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 p[4] = {
        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 0), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 1),
        __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 2), __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, 1.0f, 3)};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        v[e] = scale == 255u ? __builtin_nanf("") : ldexpf(p[e / 2][e % 2], (int)scale - 127);
}

// The casts read and write each element once and are bound by HBM: along the rows 8192 x 4096 fp16 to
// codes 17.3 us (4.9 TB/s), its codes to fp32 34.0 (4.5); down the columns 4096 x 4096 fp32 17.8 us
// (4.3 TB/s) and back 15.0 (5.1).
//
// Vectors along the rows of a [n x k] matrix: E elements to a lane, a wave to 64 E elements of a row or
// to several rows that are shorter.
struct MxRows {
    uint32_t lanes, per_row, rows;   // lanes of a vector, waves of a vector, vectors of a wave
    uint64_t waves;
};
template <int E> __host__ __device__ __forceinline__ MxRows mx_rows(uint32_t n, uint32_t k) {
    MxRows r;
    r.lanes = mx_pad(k) / E;
    r.per_row = (r.lanes + 63) / 64;
    r.rows = r.lanes < 64 ? 64 / r.lanes : 1;
    r.waves = (uint64_t)mx_ceil(n, r.rows) * r.per_row;
    return r;
}
// For every lane that has elements of a vector use(vector, lane of the vector, what load(...) of
// these gave): the loads of U pieces before the first is used, or a wave would have a kilobyte on its
// way at a time.
template <int E, int U, class Load, class Use>
__device__ __forceinline__ void mx_each(uint32_t n, uint32_t k, Load load, Use use) {
    const MxRows r = mx_rows<E>(n, k);
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t sub = r.rows > 1 ? lane / r.lanes : 0;
    // (32-bit divisions, once for U pieces: in 64 bits and for each they took longer than the stores)
    const uint32_t waves = (uint32_t)r.waves, stride = gridDim.x * 4 * U;
    for (uint32_t w0 = (blockIdx.x * 4 + wave) * U; w0 < waves; w0 += stride) {
        decltype(load(0u, 0u)) got[U];
        uint32_t vec[U], l[U], row = w0 / r.per_row, part = w0 - row * r.per_row;
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            vec[u] = row * r.rows + sub;
            l[u] = part * 64 + lane - sub * r.lanes;
            on[u] = w0 + u < waves && sub < r.rows && l[u] < r.lanes && vec[u] < n;
            if (on[u]) got[u] = load(vec[u], l[u]);
            if (++part == r.per_row) {
                part = 0;
                ++row;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (on[u]) use(vec[u], l[u], got[u]);
        if (w0 + stride < w0) break;   // past 32 bits
    }
}

template <typename T> struct MxPiece {
    float v[8];
};
template <typename T> __global__ void __launch_bounds__(256) mx_quantise_kernel(MxCastArgs a) {
    mx_each<8, 2>(
        a.n, a.k,
        [&](uint32_t vec, uint32_t l) {
            MxPiece<T> p;
            load_row<T, 8>(reinterpret_cast<const T *>(a.values) + (uint64_t)vec * a.k, l * 8, a.k, p.v);
            return p;
        },
        [&](uint32_t vec, uint32_t l, const MxPiece<T> &p) {
            const uint32_t scale = mx_scale(mx_top4(p.v));   // a block's four lanes are here together
            const uint64_t at = (uint64_t)vec * (mx_pad(a.k) / 8) + l;
            reinterpret_cast<uint32_t *>(a.codes)[at] = mx_codes(p.v, scale);
            if ((l & 3u) == 0) a.scales[at / 4] = (uint8_t)scale;
        });
}

// 16 bytes of values to a lane, so that a wave writes 1 KB without gaps.
template <typename T> constexpr int kValues = 16 / sizeof(T);
struct MxPair {
    uint32_t codes, scale;
};
template <typename T> __global__ void __launch_bounds__(256) mx_dequantise_kernel(MxCastArgs a) {
    constexpr int E = kValues<T>;
    typedef typename std::conditional<E == 8, uint32_t, uint16_t>::type Codes;
    mx_each<E, 4>(
        a.n, a.k,
        [&](uint32_t vec, uint32_t l) {
            const uint64_t at = (uint64_t)vec * (mx_pad(a.k) / E) + l;
            return MxPair{reinterpret_cast<const Codes *>(a.codes)[at], a.scales[at / (32 / E)]};
        },
        [&](uint32_t vec, uint32_t l, const MxPair &p) {
            float v[8], o[E];
            mx_values(p.codes, p.scale, v);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = v[e];
            if (l * E < a.k) store_row<T, E>(reinterpret_cast<T *>(a.values) + (uint64_t)vec * a.k, l * E, a.k, o);
        });
}

// Vectors down the columns of a [k x n] matrix: a workgroup takes 64 CV columns by 128 rows, a wave one
// block of 32 rows, a lane CV columns next to each other (256 bytes of a row to a load); the codes go
// through LDS, so that each vector's 64 bytes are written together.  (Twice the columns: 4096 x 4096
// fp32 18.7 and 17.2 us for 17.7 and 14.9, 777 x 1531 10.4 for 3.4.)
template <typename T> constexpr int kDownCols = 4 / sizeof(T);   // columns of a lane

template <typename T> __global__ void __launch_bounds__(256) mx_quantise_down_kernel(MxCastArgs a) {
    constexpr int CV = kDownCols<T>, COLS = 64 * CV;
    typedef typename Unaligned<T, CV>::type Vec;
    __shared__ u32x4 codes[COLS][5];
    __shared__ uint8_t scales[COLS][4];
    const uint32_t kp = mx_pad(a.k), ntiles = mx_ceil(a.n, COLS);
    const uint32_t ntile = blockIdx.x % ntiles, ktile = blockIdx.x / ntiles;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t k0 = ktile * 128u + wave * 32u, n0 = ntile * COLS, col = n0 + lane * CV;
    Vec v[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        const T *p = reinterpret_cast<const T *>(a.values) + (uint64_t)(k0 + e) * a.n;
        v[e] = Vec{};
        if (k0 + e < a.k) {
            if (col + CV <= a.n)
                v[e] = *reinterpret_cast<const Vec *>(p + col);
            else
#pragma unroll
                for (int c = 0; c < CV; ++c)
                    if (col + c < a.n) v[e][c] = p[col + c];
        }
    }
#pragma unroll
    for (int c = 0; c < CV; ++c) {
        uint32_t big = 0;
#pragma unroll
        for (int e = 0; e < 32; ++e) big = max(big, magnitude((float)v[e][c]));
        const uint32_t scale = mx_scale(big);
        u32x4 o;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = (float)v[8 * q + e][c];
            o[q] = mx_codes(f, scale);
        }
        codes[lane * CV + c][wave] = o;
        scales[lane * CV + c][wave] = (uint8_t)scale;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < COLS * 4; i += 256) {
        const uint32_t vec = i >> 2, part = i & 3u;
        if (n0 + vec < a.n)
            reinterpret_cast<u32x4 *>(a.codes + (uint64_t)(n0 + vec) * (kp / 2) + ktile * 64u)[part] = codes[vec][part];
    }
    for (uint32_t vec = threadIdx.x; vec < COLS; vec += 256)
        if (n0 + vec < a.n)
            *reinterpret_cast<uint32_t *>(a.scales + (uint64_t)(n0 + vec) * (kp / 32) + ktile * 4u) =
                *reinterpret_cast<const uint32_t *>(scales[vec]);
}

template <typename T> __global__ void __launch_bounds__(256) mx_dequantise_down_kernel(MxCastArgs a) {
    constexpr int CV = kDownCols<T>, COLS = 64 * CV;
    __shared__ u32x4 codes[COLS][5];
    const uint32_t kp = mx_pad(a.k), ntiles = mx_ceil(a.n, COLS);
    const uint32_t ntile = blockIdx.x % ntiles, ktile = blockIdx.x / ntiles;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t k0 = ktile * 128u + wave * 32u, n0 = ntile * COLS, col = n0 + lane * CV;
    for (uint32_t i = threadIdx.x; i < COLS * 4; i += 256) {
        const uint32_t vec = i >> 2, part = i & 3u;
        if (n0 + vec < a.n)
            codes[vec][part] = reinterpret_cast<const u32x4 *>(a.codes + (uint64_t)(n0 + vec) * (kp / 2) + ktile * 64u)[part];
    }
    uint32_t scale[CV];
#pragma unroll
    for (int c = 0; c < CV; ++c) scale[c] = a.scales[(uint64_t)min(col + c, a.n - 1) * (kp / 32) + k0 / 32u];
    __syncthreads();
    if (col >= a.n) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float f[CV][8];
#pragma unroll
        for (int c = 0; c < CV; ++c) mx_values(codes[lane * CV + c][wave][q], scale[c], f[c]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t k = k0 + 8 * q + e;
            float o[CV];
#pragma unroll
            for (int c = 0; c < CV; ++c) o[c] = f[c][e];
            if (k < a.k) store_row<T, CV>(reinterpret_cast<T *>(a.values) + (uint64_t)k * a.n, col, a.n, o);
        }
    }
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
// and their sums are joined in LDS in the order of the waves.  16 x 4096 x 4096 fp16: 9.5 us for
// 8.9 MB of w, which is latency: a launch (4 us empty), one round of loads, one of joining.
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
// as above, fragments straight from memory to registers.  256 x 4096 x 4096 fp16 15.9 us with the
// staging, 500 x 777 x 1531 fp32 3.6 + 6.6 us: one workgroup to a CU, latency of its loads.
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
// order (mx_gemm.h).  The first `xtiles` workgroups take 64 vectors of x by 128 elements, 8 elements
// of four vectors (16 apart: a word of scales) to a thread, so that a wave reads 256 bytes of a row
// together; the others 64 vectors of w's scales by 512 elements.  Vectors and elements past the
// matrix are 0.  8192 x 4096 x 4096 fp16: 20 us of 95 (84 MB); a block of 32 to a thread, its 64
// bytes read by four loads of that thread, 26.
struct MxStageArgs {
    uint32_t m, n, k, kp, k2, xtiles;
    const void *x;
    const uint8_t *w_scales;
    uint8_t *codes, *xs, *ws;
};
template <typename T> __global__ void __launch_bounds__(256) mx_stage_kernel(MxStageArgs a) {
    const uint32_t tid = threadIdx.x, blocks = a.k2 / 32u;
    if (blockIdx.x < a.xtiles) {
        const uint32_t group = blockIdx.x / (blocks / 4u), kt = blockIdx.x % (blocks / 4u);
        const uint32_t r = tid >> 4, l = tid & 15u, e0 = kt * 128u + l * 8u;
        typedef typename Unaligned<T, 8>::type Vec;
        Vec x[4];
        const T *p = reinterpret_cast<const T *>(a.x) + (uint64_t)(group * 64u + r) * a.k + e0;
        if (group * 64u + 64u <= a.m && kt * 128u + 128u <= a.k) {
#pragma unroll
            for (int q = 0; q < 4; ++q) x[q] = *reinterpret_cast<const Vec *>(p + (uint64_t)(16u * q) * a.k);
        } else {
            // what is past a row's end belongs to the next one and is dropped; a row's last elements one
            // by one would wait for each other
            const uint64_t end = (uint64_t)a.m * a.k;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t vec = group * 64u + 16u * q + r;
                const uint64_t at = (uint64_t)vec * a.k + e0;
                x[q] = Vec{};
                if (vec < a.m && e0 < a.k) {
                    if (at + 8u <= end)
                        x[q] = *reinterpret_cast<const Vec *>(reinterpret_cast<const T *>(a.x) + at);
                    else
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (at + e < end) x[q][e] = reinterpret_cast<const T *>(a.x)[at + e];
                }
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[q][e] = e0 + e < a.k ? x[q][e] : (T)0;
        }
        uint32_t word = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (float)x[q][e];
            const uint32_t scale = mx_scale(mx_top4(v));
            word |= scale << (8 * q);
            reinterpret_cast<uint32_t *>(a.codes)[(uint64_t)(group * 64u + 16u * q + r) * (a.k2 / 8u) + e0 / 8u] =
                mx_codes(v, scale);
        }
        if ((l & 3u) == 0) reinterpret_cast<uint32_t *>(a.xs)[((uint64_t)group * blocks + kt * 4u + l / 4u) * 16u + r] = word;
        return;
    }
    __shared__ uint8_t bytes[16][64];   // block, then 4 r + q of vector 16 q + r
    const uint32_t quads = (blocks + 15u) / 16u, tile = blockIdx.x - a.xtiles, group = tile / quads, b0 = tile % quads * 16u;
    const uint32_t vec = tid >> 2, b = b0 + (tid & 3u) * 4u;
    uint32_t four = 0;
    if (group * 64u + vec < a.n && b < a.kp / 32u)   // (kp / 32 is a multiple of 4)
        four = *reinterpret_cast<const uint32_t *>(a.w_scales + (uint64_t)(group * 64u + vec) * (a.kp / 32u) + b);
#pragma unroll
    for (int c = 0; c < 4; ++c) bytes[(tid & 3u) * 4u + c][(vec & 15u) * 4u + (vec >> 4)] = (uint8_t)(four >> (8 * c));
    __syncthreads();
    if (b0 + (tid >> 4) < blocks)
        reinterpret_cast<uint32_t *>(a.ws)[((uint64_t)group * blocks + b0) * 16u + tid] = reinterpret_cast<const uint32_t *>(bytes)[tid];
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
    a.k2 = st.k2 = (uint32_t)w.k2;
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
    a.tiles_m = mx_ceil(f.m, BT);
    a.tiles_n = mx_ceil(f.n, BT);
    st.xtiles = (uint32_t)mx_stage_x(w);
    hipLaunchKernelGGL(mx_stage_kernel<T>, dim3((uint32_t)mx_stage_groups(w)), dim3(256), 0, s, st);
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
        hipLaunchKernelGGL((mx_rows_kernel<T, 1, U>), dim3(mx_ceil(a.n, 16)), dim3(512), 0, s, a);
    else
        hipLaunchKernelGGL((mx_rows_kernel<T, 2, U / 2>), dim3(mx_ceil(a.n, 16)), dim3(512), 0, s, a);
    return hipGetLastError();
}

template <typename T> hipError_t mx_cast(const MxCastArgs &a, bool down, bool back, hipStream_t s) {
    if (a.n == 0 || a.k == 0) return hipSuccess;
    if (down) {
        constexpr uint32_t cols = mx_down_cols(sizeof(T));
        static_assert(cols == 64 * kDownCols<T>, "what the kernels take");
        const dim3 grid(mx_ceil(a.n, cols) * (mx_pad(a.k) / 128));
        hipLaunchKernelGGL((back ? mx_dequantise_down_kernel<T> : mx_quantise_down_kernel<T>), grid, dim3(256), 0, s, a);
    } else {
        const uint64_t waves = back ? mx_rows<kValues<T>>(a.n, a.k).waves : mx_rows<8>(a.n, a.k).waves;
        // workgroups that loop: 8192 x 4096 fp16 to codes 17.4 us on 2048, 20.2 on one per piece; its
        // values to fp32 34.0 us on 4096, 41.6
        const uint64_t groups = (waves + 3) / 4, most = back ? 4096 : 2048;
        const dim3 grid((uint32_t)(groups < most ? groups : most));
        hipLaunchKernelGGL((back ? mx_dequantise_kernel<T> : mx_quantise_kernel<T>), grid, dim3(256), 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_quantise(const MxCastArgs &a, uint32_t dtype, bool down, hipStream_t s) {
    return dtype ? mx_cast<half_t>(a, down, false, s) : mx_cast<float>(a, down, false, s);
}

hipError_t launch_mx_dequantise(const MxCastArgs &a, uint32_t dtype, bool down, hipStream_t s) {
    return dtype ? mx_cast<half_t>(a, down, true, s) : mx_cast<float>(a, down, true, s);
}

hipError_t launch_mx_forward(const MxForwardArgs &a, uint32_t dtype, hipStream_t s) {
    return dtype ? mx_forward_t<half_t>(a, s) : mx_forward_t<float>(a, s);
}

}  // namespace skl

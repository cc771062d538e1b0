// ffn_rows.hip — the forward products of ffn.h for up to 64 rows (gfx950): a stream over the weights.
//
// k goes in up to eight slices, each to an XCD or to neighbours that halve its columns (workgroup L runs
// on XCD L % 8), so that an XCD reads whole or half rows of W [k x n]; within a slice a workgroup owns 16 VN
// columns of each matrix of a pair and its waves share the slice's k, 32 k (fp16) or 16 k (fp32) to a step.
// With eight slices 256 workgroups are in flight from 4096 columns on (VN 8; VN 4: 2048), and fewer below:
// 64 of 1024 columns.  The weights go from memory to registers as they are stored, VN columns of a k-row to a
// lane, 16 lanes to the row.  fp16
// lanes turn 8 k-rows into fragments by permutes, one MFMA (16x16x32) for each of their VN columns,
// whose n index is then VN (lane % 16) + j; fp32 lanes hold a fragment (16x16x4) as loaded.  The waves'
// sums are added in LDS, the slices' by a second launch, both in a fixed order, in front of the epilogue.
//
// What bounds it: HBM, the weights read once (floor at the 5.12 TB/s of a copy).  One row, weights from
// memory, the K-splitting kernel's tiles of 16 to 64 columns over all of k in brackets, where each XCD has
// a narrow strip of every row and few waves share a long k: pair fp16 8192 x 4096 30 us (63; floor 26),
// 4096 x 8192 29 (36; 26), 11008 x 4096 37 (83; 35), 3000 x 3000 14 (21; 7), 4096 x 1024 13 (27; 3); fp32
// 4096 x 8192 52 (66; 52); projection fp16 8192 x 4096 18 (28; 13), 3000 x 3000 9.3 (10; 3.5).  Narrower layers
// stay 2 to 4 times over the floor: too few workgroups for the memory, and 3 to 4 us of the second launch.  For
// that launch the other kernel is ahead where k is short (product_rows_size), and it can be where caches hold
// the weights (pair 4096 x 1024, called again at once: 9.6 and 7.5), which a network's layers between two
// calls do not leave there.
// 17 to 32 rows have two blocks of rows to a fragment of the weights, more have four; fp16 lanes then own 4
// columns, as the sums of 8 would not leave registers for the loads ahead.  32 rows: pair fp16 8192 x 4096
// 37 (69), 4096 x 8192 33 (38), 11008 x 4096 45 (93), fp32 4096 x 8192 61 (75); projection fp16 8192 x 4096
// 22 (38), 4096 x 1024 9.4 (14).  64 rows, fp16: pair 8192 x 4096 42 (74), 4096 x 8192 39 (41), projection
// 8192 x 4096 27 (35).
#include "ffn.h"
#include "ffn_epi.h"
#include "gemm.h"

namespace skl {

constexpr uint32_t kSlices = 8;   // the most
constexpr uint32_t kOut = 0x80000000u;   // an offset past every operand: reads as zero

template <int N> struct Words { typedef uint32_t type __attribute__((ext_vector_type(N))); };

template <int N> __device__ __forceinline__ typename Words<N>::type rows_load(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    if constexpr (N == 2) return __builtin_bit_cast(typename Words<2>::type, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0));
    else return __builtin_bit_cast(typename Words<4>::type, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}

// The weights of one step of one matrix: L loads of VN columns, fp16 k-rows 8 (lane / 16) + i,
// fp32 k-rows 4 i + lane / 16.
template <typename T, int VN> struct RowsW {
    static constexpr int L = sizeof(T) == 2 ? 8 : 4;
    static constexpr int NW = VN * (int)sizeof(T) / 4;   // words of a load
    typename Words<NW>::type v[L];
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t row) {
#pragma unroll
        for (int i = 0; i < L; ++i) v[i] = rows_load<NW>(r, off + (sizeof(T) == 2 ? i : 4 * i) * row);
    }
    // fp16: the fragment of the lane's column j, its 8 k
    __device__ __forceinline__ u32x4 frag(int j) const {
        const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
        u32x4 f;
#pragma unroll
        for (int p = 0; p < 4; ++p) f[p] = __builtin_amdgcn_perm(v[2 * p + 1][j >> 1], v[2 * p][j >> 1], sel);
        return f;
    }
};

// x of one step, row lane % 16: fp16 k 8 (lane / 16) .. + 7, fp32 k 4 i + lane / 16, i < 4.
template <typename T> struct RowsX {
    u32x4 v;
    // left: k of the row from the step's first on (fp16: from the lane's first); past it zeros, as the bytes there
    // are the next row's
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, uint32_t off, int left) {
        if constexpr (sizeof(T) == 2) {
            v = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)(left > 0 ? off : kOut), 0, 0));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)(left > 4 * i ? off + 16 * i : kOut), 0, 0);
        }
    }
};

// planes: [sh.k_per_split slices][P][M][N] fp32
template <typename T, int P, int VN, int MB, int W, int D>
__global__ void __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(W / 4, W / 4)))
    rows_kernel(GemmShape sh, const T *__restrict__ A, const T *__restrict__ B, const T *__restrict__ B2, float *planes) {
    constexpr uint32_t CW = 16 * VN, KS = sizeof(T) == 2 ? 32 : 16, NT = 64 * W, EP = CW + 4, BM = 16 * MB;
    __shared__ __attribute__((aligned(16))) float E[W * BM * EP];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // XCDs 8 / slices to a slice, each with a contiguous part of its column groups
    const uint32_t share = 8u / sh.k_per_split, slice = blockIdx.x % 8u / share, groups = (sh.N + CW - 1) / CW;
    const uint32_t mine = (groups + share - 1) / share, group = blockIdx.x % share * mine + blockIdx.x / 8u;
    if (blockIdx.x / 8u >= mine || group >= groups) return;
    const uint32_t n0 = group * CW, g = lane >> 4, c = lane & 15u;
    const uint32_t all = (sh.K + KS - 1) / KS, per = (all + sh.k_per_split - 1) / sh.k_per_split;
    const uint32_t first = min(slice * per, all), end = min(first + per, all);

    const uint32_t wbytes = sh.K * sh.ldb * (uint32_t)sizeof(T), row = sh.ldb * (uint32_t)sizeof(T);
    __amdgpu_buffer_rsrc_t rw[P], rx;
    rw[0] = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(B), (short)0, (int)wbytes, 0x00020000);
    if constexpr (P == 2) rw[1] = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(B2), (short)0, (int)wbytes, 0x00020000);
    rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(A), (short)0, (int)(((sh.M - 1) * sh.lda + sh.K) * (uint32_t)sizeof(T)),
                                           0x00020000);
    // k-row of the lane's first load; columns past the last are not read
    const uint32_t krow = sizeof(T) == 2 ? 8u * g : g, ncol = n0 + VN * c;
    const uint32_t woff = ncol < sh.N ? krow * row + ncol * (uint32_t)sizeof(T) : kOut;
    uint32_t xoff[MB];
#pragma unroll
    for (uint32_t i = 0; i < MB; ++i) {
        const uint32_t m = 16 * i + c;
        xoff[i] = m < sh.M ? (m * sh.lda + krow) * (uint32_t)sizeof(T) : kOut;
    }

    floatx4 acc[P][VN][MB];
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int j = 0; j < VN; ++j)
#pragma unroll
            for (int i = 0; i < MB; ++i) acc[p][j][i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

    RowsW<T, VN> w[D][P];
    RowsX<T> x[D][MB];
    auto load = [&](int d, uint32_t s) {   // steps past the slice's last read zeros on both sides, as do k past K
        const uint32_t k0 = s * KS;
        const bool in = s < end;
#pragma unroll
        for (int p = 0; p < P; ++p) w[d][p].load(rw[p], in && woff != kOut ? woff + k0 * row : kOut, row);
#pragma unroll
        for (int i = 0; i < MB; ++i)
            x[d][i].load(rx, xoff[i] + k0 * (uint32_t)sizeof(T),
                         in && xoff[i] != kOut ? (int)sh.K - (int)(k0 + (sizeof(T) == 2 ? krow : 0u)) : 0);
    };
    auto work = [&](int d) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int j = 0; j < VN; ++j) {
                    const halfx8 f = __builtin_bit_cast(halfx8, w[d][p].frag(j));
#pragma unroll
                    for (int i = 0; i < MB; ++i)
                        acc[p][j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, __builtin_bit_cast(halfx8, x[d][i].v),
                                                                              acc[p][j][i], 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int p = 0; p < P; ++p)
#pragma unroll
                    for (int j = 0; j < VN; ++j)
#pragma unroll
                        for (int i = 0; i < MB; ++i)
                            acc[p][j][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __builtin_bit_cast(float, (uint32_t)w[d][p].v[q][j]),
                                __builtin_bit_cast(float, (uint32_t)x[d][i].v[q]), acc[p][j][i], 0, 0, 0);
        }
    };
#pragma unroll
    for (int d = 0; d < D; ++d) load(d, first + wave + d * W);
    for (uint32_t s = first + wave; s < end; s += D * W) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            work(d);
            load(d, s + (D + d) * W);
        }
    }
    // lane l, register r of block (j, i): row 16 i + l % 16, column VN (4 (l / 16) + r) + j
#pragma unroll
    for (int p = 0; p < P; ++p) {
        if (p) lds_barrier();
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < VN; j += 4)
                    *reinterpret_cast<floatx4 *>(E + (wave * BM + 16 * i + c) * EP + VN * (4 * g + r) + j) =
                        floatx4{acc[p][j][i][r], acc[p][j + 1][i][r], acc[p][j + 2][i][r], acc[p][j + 3][i][r]};
        lds_barrier();
        for (uint32_t q = tid; q < BM * CW / 4; q += NT) {
            const uint32_t m = q / (CW / 4), cc = (q % (CW / 4)) * 4, n = n0 + cc;
            if (m >= sh.M || n >= sh.N) continue;
            floatx4 v = *reinterpret_cast<const floatx4 *>(E + m * EP + cc);
#pragma unroll
            for (int k = 1; k < W; ++k) v += *reinterpret_cast<const floatx4 *>(E + (k * BM + m) * EP + cc);
            *reinterpret_cast<floatx4 *>(planes + ((uint64_t)(slice * P + p) * sh.M + m) * sh.N + n) = v;
        }
    }
}

// The sums of the S slices' planes, 4 columns to a thread, and the epilogue.
template <class Epi, int P, int S>
__global__ void __launch_bounds__(64) rows_join_kernel(GemmShape sh, const float *planes, typename Epi::Params ep) {
    const uint32_t per = sh.N / 4, q = blockIdx.x * 64 + threadIdx.x, m = q / per, n = q % per * 4;
    if (m >= sh.M) return;
    floatx4 v[S][P];
#pragma unroll
    for (uint32_t s = 0; s < S; ++s)
#pragma unroll
        for (int p = 0; p < P; ++p)
            v[s][p] = *reinterpret_cast<const floatx4 *>(planes + ((uint64_t)(s * P + p) * sh.M + m) * sh.N + n);
    const uint64_t idx = (uint64_t)m * Epi::ldc(ep) + n;
    typename EpiReadsPre<Epi, EpiReads<Epi>::value>::Pre pre;
    if constexpr (EpiReads<Epi>::value) Epi::load(ep, idx, m, pre);
    const typename Epi::Col col = Epi::column(ep, n);
#pragma unroll
    for (uint32_t s = 1; s < S; ++s)
#pragma unroll
        for (int p = 0; p < P; ++p) v[0][p] += v[s][p];
    if constexpr (P == 2)
        Epi::finish(ep, idx, v[0][0], v[0][1], col);
    else
        Epi::finish(ep, idx, m, n, v[0][0], col, pre);
}

// Columns of a lane: 16 bytes of them, half of that where fp16 has two blocks of rows to sum for.
static uint32_t rows_vn(uint32_t dtype, uint32_t M) { return dtype == 1 && M <= 16 ? 8 : 4; }
// Slices of k: as many as 256 workgroups allow.
static uint32_t rows_slices(uint32_t dtype, uint32_t M, uint32_t N) {
    const uint32_t cw = 16 * rows_vn(dtype, M), groups = (N + cw - 1) / cw;
    return groups <= 32 ? 8 : groups <= 64 ? 4 : groups <= 128 ? 2 : 1;
}

size_t product_rows_bytes(uint32_t M, uint32_t N, uint32_t matrices) {
    return (size_t)kSlices * matrices * M * N * sizeof(float);
}

// Where the two launches are ahead of the K-splitting kernel's one: k long enough for eight slices of it (that
// kernel's 16x16 tiles take a step more behind every 1024 k, a pair's behind every 512, and so it loses what it
// was ahead in some places).  Both measured with weights from memory, k of 512 to 16384 and 64 to 8192 columns (us, the
// K-splitting kernel behind the stroke).  Short k are ahead only for a pair of enough columns:
//   one row     fp16 pair 3008 x 64 8.7/9.4, 2048 x 256 9.1/8.3, 2904 x 256 9.9/12.1, 2048 x 512 10.9/14.2, 1504 x 512
//               8.9/7.6, 1504 x 1024 10.6/10.8; fp32 pair 2048 x 64 8.3/8.5, 1504 x 256 9.0/9.4, 1024 x 1024 9.6/10.2
//               projection fp16 3008 x 64 6.4/6.7, 2048 x 512 6.9/5.9, fp32 3008 x 64 7.5/8.0
// Past 16 rows the sums of the blocks of rows take more of the registers, and the fp32 MFMAs bound one matrix
// (4096 x 8192, 32 rows: 42/30); past 32 rows four blocks have registers in fp16 only:
//   32 rows     fp16 pair 3008 x 256 10.5/11.4, 2048 x 1024 12.6/13.5, 1504 x 8192 19.0/17.3; fp32 pair 3008 x 256
//               19.6/20.7, 2048 x 4096 24.2/22.1; fp16 projection 3480 x 264 8.1/9.6, 3008 x 512 8.2/7.3, 3008 x 1024 9.6/10.8
//   64 rows     fp16 pair 3880 x 384 13.7/16.2, 3008 x 256 12.7/10.4, 3008 x 512 14.9/17.4; projection 8192 x 256
//               14.0/18.9, 4096 x 2048 13.8/18.2, 4096 x 1024 11.9/12.3, 3008 x 4096 16.5/15.0
bool product_rows_size(uint32_t dtype, uint32_t M, uint32_t N, uint32_t K, uint32_t matrices) {
    const bool half = dtype == 1, pair = matrices == 2;
    const uint64_t t = half ? 2 : 4;
    const uint32_t lane = half ? 8 : 4;
    bool ahead = false;
    if (M <= 16)
        ahead = N >= 64 && (K >= 3000 || (pair && (half ? (K >= 1500 && (uint64_t)K * N >= 1u << 20) || (K >= 2100 && N >= 256)
                                                        : K >= 2000 || (K >= 1500 && N >= 256))));
    else if (M <= 32 && pair)
        ahead = N >= 256 && (K >= 3000 || (half && K >= 2000 && N >= 512));
    else if (M <= 32)
        ahead = half && N >= 256 && K >= (N >= 1000 ? 3000 : 3100);
    else if (M <= 64 && half)
        ahead = pair ? N >= 256 && K >= (N >= 512 ? 3000 : 3100)
                     : N >= 256 && (K >= 8000 || (K >= 4000 && N >= 2000));
    return M && ahead && N % lane == 0 && K % lane == 0 && (K + 64ull) * N * t < (1ull << 31);
}

bool product_rows_ok(const ProductLaunch &p) {
    const GemmLaunch &g = p.g;
    if (p.kind != Product::Pair && p.kind != Product::Project) return false;
    const bool pair = p.kind == Product::Pair;
    const uint64_t t = g.dtype == 1 ? 2 : 4;
    auto on = [](const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
    return product_rows_size(g.dtype, g.M, g.N, g.K, pair ? 2 : 1) && on(g.A) && g.lda * t % 16 == 0 &&
           (uint64_t)g.M * g.lda * t < (1ull << 31) && on(g.B) && (!pair || on(p.pair.b2)) && product_rows4(p);
}

template <typename T, class Epi, int MB>
static hipError_t rows_mb(const ProductLaunch &p, const typename Epi::Params &e, float *planes, hipStream_t s) {
    constexpr int P = EpiPair<Epi>::value ? 2 : 1, VN = sizeof(T) == 2 && MB == 1 ? 8 : 4, W = 8, D = 2;
    GemmShape sh{};
    sh.M = p.g.M;
    sh.N = p.g.N;
    sh.K = p.g.K;
    sh.lda = p.g.lda;
    sh.ldb = p.g.ldb;
    const T *b2 = nullptr;
    if constexpr (P == 2) b2 = reinterpret_cast<const T *>(e.b2);
    sh.k_per_split = rows_slices(p.g.dtype, sh.M, sh.N);
    const uint32_t share = 8 / sh.k_per_split, groups = (sh.N + 16 * VN - 1) / (16 * VN);
    launch_timed(p.g, rows_kernel<T, P, VN, MB, W, D>, dim3((groups + share - 1) / share * 8), dim3(64 * W), s, sh,
                 reinterpret_cast<const T *>(p.g.A), reinterpret_cast<const T *>(p.g.B), b2, planes);
    const dim3 join((uint32_t)(((uint64_t)sh.M * (sh.N / 4) + 63) / 64));
    switch (sh.k_per_split) {
    case 8: rows_join_kernel<Epi, P, 8><<<join, 64, 0, s>>>(sh, planes, e); break;
    case 4: rows_join_kernel<Epi, P, 4><<<join, 64, 0, s>>>(sh, planes, e); break;
    case 2: rows_join_kernel<Epi, P, 2><<<join, 64, 0, s>>>(sh, planes, e); break;
    default: rows_join_kernel<Epi, P, 1><<<join, 64, 0, s>>>(sh, planes, e);
    }
    return hipGetLastError();
}

template <typename T, class Epi>
static hipError_t rows_t(const ProductLaunch &p, const typename Epi::Params &e, float *planes, hipStream_t s) {
    if constexpr (sizeof(T) == 2 || EpiPair<Epi>::value)
        if (p.g.M > 16 && p.g.M <= 32) return rows_mb<T, Epi, 2>(p, e, planes, s);
    if constexpr (sizeof(T) == 2)
        if (p.g.M > 32) return rows_mb<T, Epi, 4>(p, e, planes, s);
    return rows_mb<T, Epi, 1>(p, e, planes, s);
}

hipError_t launch_product_rows(const ProductLaunch &p, void *work, hipStream_t s) {
    if (!product_rows_ok(p)) return hipErrorInvalidValue;
    float *planes = reinterpret_cast<float *>(work);
    if (p.g.dtype == 1) {
        if (p.kind == Product::Pair) return rows_t<half_t, EpiPairK<half_t>>(p, p.pair, planes, s);
        return p.stream_dtype == 1 ? rows_t<half_t, EpiProjectK<half_t, half_t>>(p, p.project, planes, s)
                                   : rows_t<half_t, EpiProjectK<half_t, float>>(p, p.project, planes, s);
    }
    return p.kind == Product::Pair ? rows_t<float, EpiPairK<float>>(p, p.pair, planes, s)
                                   : rows_t<float, EpiProjectK<float, float>>(p, p.project, planes, s);
}

}  // namespace skl

// mx_gemm.h — the product of two MXFP4 matrices on 256x256 or 128x128 tiles, gfx950.
//
// out [m x n] = act(X . W^T + bias): X and W as vectors of k elements, codes k-contiguous.  A
// k-tile is 256 elements, 128 bytes of each of a tile's vectors: the bytes, and the matrix
// instructions' cycles, of a 64-element k-tile of an fp16 product, so operands are staged as that
// kernel's are (gemm_dma.h, OpK): two stages in LDS, filled by loads that go there directly, the
// 16-byte chunk c of vector r at slot c ^ (r / 2 % 8), which is one block of 32 elements, and a
// fragment (16 vectors by 128 elements) is one ds_read_b128 per lane.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes the scale of a lane's block (vector lane % 16, block
// lane / 16 of the step) from one byte of a register, which one chosen by the instruction.  The
// scales are staged so that the four bytes are those of four fragments: per 64 vectors and block,
// 16 words, word r holding vectors r, r + 16, r + 32 and r + 48.  One ds_read_b32 then feeds four
// fragments.
#pragma once

#include "gemm_dma.h"
#include "mxfp4.h"
#include "rows.h"

// 8192 x 4096 x 4096 fp16 with SiLU: 75 us, 3.7 PFLOP/s, behind 20 of staging.  Per 4096 of k 53 us:
// 40 with neither loads nor LDS reads in the loop (MFMAs and barriers), 46 without the reads, 49
// without the loads; loads early in their step or a raised wave priority around the MFMAs do not
// change it.  The other 22 us are the epilogues (activations on the VALU, 67 MB of stores) and the
// start of each of two rounds of tiles.
namespace skl {

typedef int intx8 __attribute__((ext_vector_type(8)));

// acc += w x: block codes w and x with scale bytes WB of ws and XB of xs.  In asm, the accumulator in
// AGPRs and in place: left to the compiler 128 accumulators are moved about and spill.  Its hazard
// checks do not look in here, so the kernel keeps VALU writes of these registers out of the loop
// and waits before it reads the sums.
template <int WB, int XB>
__device__ __forceinline__ void mx_mma(f32x4 &acc, const u32x4 &w, uint32_t ws, const u32x4 &x, uint32_t xs) {
    asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%6,0] op_sel_hi:[%7,%8,0] cbsz:4 blgp:4"
                 : "+a"(acc)
                 : "v"(w), "v"(x), "v"(ws), "v"(xs), "i"(WB & 1), "i"(XB & 1), "i"(WB >> 1), "i"(XB >> 1));
}

template <int OFF> __device__ __forceinline__ void ds_read4(uint32_t &dst, uint32_t addr) {
    asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(dst) : "v"(addr), "i"(OFF) : "memory");
}
__device__ __forceinline__ void pin(uint32_t &v) { asm volatile("" : "+v"(v)); }

template <int F> struct Each {   // f(0), f(1), ... as constants
    template <class Fn> __device__ __forceinline__ static void run(Fn f) {
        Each<F - 1>::run(f);
        f(std::integral_constant<int, F - 1>());
    }
};
template <> struct Each<0> {
    template <class Fn> __device__ __forceinline__ static void run(Fn) {}
};

// The activation of several values, chosen once for them; the fast forms of device_math.h, a few
// units in the last place of fp32 each.
template <int N> __device__ __forceinline__ void activate(uint32_t act, float leaky, float (&v)[N]) {
    auto each = [&](auto f) {
#pragma unroll
        for (int c = 0; c < N; ++c) v[c] = f(v[c]);
    };
    switch (act) {
    case 1: each([](float x) { return sigmoid_fast(x); }); break;
    case 2: each([](float x) { return fmaxf(0.0f, x); }); break;
    case 3: each([&](float x) { return x > 0.0f ? x : leaky * x; }); break;
    case 4: each([](float x) { return tanh_fast(x); }); break;
    case 6: each([](float x) { return x * sigmoid_fast(x); }); break;
    case 7: each([](float x) { return mish_fast(x); }); break;
    default: break;
    }
}

struct MxGemmArgs {
    uint32_t m, n, kp, k2;          // kp: W's padded k; k2: of X's codes and both scales, a multiple of 256
    uint32_t tiles_m, tiles_n;
    const uint8_t *x, *xs, *w, *ws;   // X codes [.. x k2 / 2]; staged scales; W codes [n x kp / 2]; staged scales
    const void *bias;
    uint32_t act;
    float leaky;
    void *out;
};

// BT: tile edge.  256: eight waves, two to a SIMD, each 128 x 64 of the tile; X's fragments are read
// in place, each behind its last MFMA, as 128 accumulators leave no room for two sets.  128: four
// waves of 64 x 64, two workgroups to a CU, both operands' fragments double.  (256 on four waves of
// 128 x 128 with double fragments has the faster k loop, 51 us per 4096 of k over 8192 x 4096 against
// 53, but one wave per SIMD hides nothing in the epilogue: 8192 x 4096 x 4096 with SiLU 82 us
// against 78.)
template <typename T, int BT>
__global__ void __launch_bounds__(2 * BT) __attribute__((amdgpu_waves_per_eu(2, 2))) mx_gemm_kernel(MxGemmArgs a) {
    constexpr int NW = BT / 32, WN = BT / 64, TWM = BT / 2, MT = TWM / 16, NTL = 4;
    constexpr int MG = MT / 4;                          // scale words of a wave's X fragments; W's: one
    constexpr int OP = BT * 128, SC = BT / 64 * 512;    // bytes of an operand's codes and scales per stage
    constexpr int STAGE = 2 * OP + 2 * SC;
    constexpr int IPO = BT / 8 / NW;                    // 1 KB loads of a wave per operand and tile
    constexpr int SLOADS = 2 * SC / 1024;               // of the whole workgroup for the scales
    constexpr bool kInPlace = BT == 256;
    static_assert(SLOADS <= NW && SC % 1024 == 0, "at most one scale load per wave");
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
    lds_char *lsm = (lds_char *)(smem);
    const uint32_t tid = threadIdx.x, lane = tid & 63u, r = lane & 15u, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wm = wave / WN, wn = wave % WN;
    uint32_t tm, tn;
    tile_coords(blockIdx.x, a.tiles_m, a.tiles_n, tm, tn);
    const uint32_t m0 = tm * BT, n0 = tn * BT;
    const int nk = (int)(a.k2 / 256u);

    // loads: instruction t of a wave fills vectors 8 (NW t + wave) .. + 7 of the tile; X has whole
    // tiles of vectors, W's past its end read the last one (not stored)
    const uint32_t row0 = 8u * wave + (lane >> 3), kc = (lane & 7u) ^ ((row0 >> 1) & 7u);
    const uint32_t xp = a.k2 / 2, wp = a.kp / 2;
    const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t *>(a.x + (uint64_t)m0 * xp), (short)0, (int)0xffffffff, 0x00020000);
    const __amdgpu_buffer_rsrc_t wr =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(a.w + (uint64_t)n0 * wp), (short)0, (int)0xffffffff, 0x00020000);
    const uint32_t xo = row0 * xp + kc * 16u, wlast = a.n - 1u - n0;
    // W's last k-tile may be half there: its upper chunks are read from the lower half (X's codes
    // are zero against them)
    const bool half = a.kp % 256u;
    // scales: load q of SLOADS fills 1 KB, two groups of 64 vectors with 8 blocks each; wave q's
    const uint32_t sq = wave % SLOADS, sg = (sq * 2u + lane / 32u) % (BT / 64u);
    const bool s_is_w = sq * 2u >= BT / 64u;
    const uint8_t *sp = (s_is_w ? a.ws + (uint64_t)(n0 / 64u) * (a.k2 * 2u) : a.xs + (uint64_t)(m0 / 64u) * (a.k2 * 2u));
    const __amdgpu_buffer_rsrc_t sr =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(sp), (short)0, (int)0xffffffff, 0x00020000);
    const uint32_t so = sg * (a.k2 * 2u) + (lane % 32u) * 16u;
    auto dma = [&](const __amdgpu_buffer_rsrc_t &rs, uint32_t off, uint32_t add, lds_char *to) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, reinterpret_cast<__attribute__((address_space(3))) void *>(to), 16,
                                                 (int)off, (int)add, 0, 0);
    };
    // load q of this wave for k-tile kt
    auto load = [&](int kt, uint32_t stage, int q) {
        lds_char *st = lsm + stage;
        if (q < IPO) {
            dma(xr, xo, (uint32_t)kt * 128u + (uint32_t)q * 8u * NW * xp, st + (NW * q + wave) * 1024u);
        } else if (q < 2 * IPO) {
            // (made anew each time: four registers more would spill)
            uint32_t v = row0;
            asm volatile("" : "+v"(v));
            const uint32_t chunk = half && kt + 1 == nk ? kc & 3u : kc;
            dma(wr, min(v + 8u * NW * (uint32_t)(q - IPO), wlast) * wp + chunk * 16u, (uint32_t)kt * 128u,
                st + OP + (NW * (q - IPO) + wave) * 1024u);
        } else if (wave < SLOADS)
            dma(sr, so, (uint32_t)kt * 512u, st + 2 * OP + sq * 1024u);
    };

    f32x4 acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) {
            acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            asm volatile("s_nop 1" : "+a"(acc[i][j]));   // two wait states before its first use
        }

    const uint32_t lds0 = (uint32_t)(uintptr_t)lsm, swz = g ^ ((r >> 1) & 7u);
    const uint32_t xf = lds0 + (wm * TWM + r) * 128u, wf = lds0 + OP + (wn * 64u + r) * 128u;
    const uint32_t xsf = lds0 + 2 * OP + wm * MG * 512u + g * 64u + r * 4u;
    const uint32_t wsf = lds0 + 2 * OP + SC + wn * 512u + g * 64u + r * 4u;
    u32x4 fx[kInPlace ? 1 : 2][MT], fw[2][NTL];
    uint32_t sx[2][MG], sw[2];
    constexpr int NDMA = 2 * IPO + 1;
    // W's fragments and both scales of step KS of the tile in `stage`, into set KS; X's fragment I
    auto read_w = [&](uint32_t stage, auto ks) {
        constexpr int KS = decltype(ks)::value;
        const uint32_t at = wf + stage + ((4u * KS) ^ swz) * 16u;
        Each<NTL>::run([&](auto j) { ds_read16<decltype(j)::value * 2048>(fw[KS][j], at); });
        ds_read4<KS * 256>(sw[KS], wsf + stage);
        Each<MG>::run([&](auto q) { ds_read4<decltype(q)::value * 512 + KS * 256>(sx[KS][q], xsf + stage); });
    };
    auto read_x = [&](auto i, uint32_t stage, auto ks) {
        constexpr int KS = decltype(ks)::value;
        ds_read16<decltype(i)::value * 2048>(fx[kInPlace ? 0 : KS][i], xf + stage + ((4u * KS) ^ swz) * 16u);
    };
    auto pin_w = [&](auto ks) {
        constexpr int KS = decltype(ks)::value;
#pragma unroll
        for (int j = 0; j < NTL; ++j) pin(fw[KS][j]);
        pin(sw[KS]);
#pragma unroll
        for (int q = 0; q < MG; ++q) pin(sx[KS][q]);
    };
    auto pin_x = [&](auto ks) {
#pragma unroll
        for (int i = 0; i < MT; ++i) pin(fx[kInPlace ? 0 : decltype(ks)::value][i]);
    };
    typedef std::integral_constant<int, 0> Zero;
    typedef std::integral_constant<int, 1> One;
    // LDS reads complete in order.  Before row 0 of a step the reads behind X's fragment 0 may be
    // pending, the other MT - 1; before row i > 0 the rest of those and what rows 0 .. i - 1 issued.
    constexpr int W0 = MT - 1, W1 = MT - 1 + NTL + 1 + MG;
    static_assert(W1 <= 15, "the counter's range");
    // Step KS: row by row of X's fragments its MFMAs, then the reads of the step after it (of the
    // tile in `from`) and, in the second step, the loads of k-tile kn into `to`.  X's fragment I is
    // read behind its own row (in place) or the row before it.
    auto step = [&](auto ks, uint32_t from, int kn, uint32_t to) {
        constexpr int KS = decltype(ks)::value;
        typedef std::integral_constant<int, 1 - KS> Next;
        Each<MT>::run([&](auto i) {
            constexpr int I = decltype(i)::value;
            if constexpr (KS == 0) {
                if constexpr (!kInPlace) {
                    if constexpr (I == 0) {
                        wait_lgkmcnt<0>();
                        pin_w(ks);
                        pin_x(ks);
                    }
                } else if constexpr (I == 0) {
                    wait_lgkmcnt<W0>();
                    pin_w(ks);
                    pin(fx[0][0]);
                } else {
                    wait_lgkmcnt<W1>();
                    pin(fx[0][I]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            Each<NTL>::run([&](auto j) {
                mx_mma<decltype(j)::value, I % 4>(acc[I][j], fw[KS][j], sw[KS], fx[kInPlace ? 0 : KS][I], sx[KS][I / 4]);
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr (KS == 1)
#pragma unroll
                for (int q = I * NDMA / MT; q < (I + 1) * NDMA / MT; ++q) load(kn, to, q);
            if constexpr (I == 0) read_w(from, Next());
            read_x(i, from, Next());
            __builtin_amdgcn_sched_barrier(0);
        });
    };

#pragma unroll
    for (int q = 0; q < NDMA; ++q) load(0, 0, q);
    wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int q = 0; q < NDMA; ++q) load(min(1, nk - 1), STAGE, q);
    read_w(0u, Zero());
    Each<MT>::run([&](auto i) { read_x(i, 0u, Zero()); });
    uint32_t stage = 0;
    for (int kt = 0; kt < nk; ++kt) {
        step(Zero(), stage, 0, 0u);
        // the next tile has landed, and every read of this one's stage is done
        wait_vmcnt<0>();
        wait_lgkmcnt<0>();
        pin_w(One());
        pin_x(One());
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        const uint32_t other = STAGE - stage;
        // past the end: the last tile again, not used
        step(One(), other, min(kt + 2, nk - 1), stage);
        stage = other;
    }
    wait_vmcnt<0>();
    wait_lgkmcnt<0>();
    pin_w(Zero());
    pin_x(Zero());
    // wait states before the last sums are read (and those reads stay below)
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j) asm volatile("" : "+a"(acc[i][j]));

    // Epilogue, from the registers: a lane's block holds columns 16 j + 4 g .. + 3 of row 16 i + r.
    // For fp16 the lanes of two neighbouring g exchange halves of two blocks, so that each has 8
    // columns of one, and an instruction stores 16 rows by 64 bytes.  A loop over the rows of blocks,
    // with the accumulators (whose registers are fixed) taken by a switch: unrolled, the activations
    // would be 300 KB of code for a 64 KB instruction cache.
    const uint32_t nw = n0 + wn * 64u;
    float bias[NTL * 4];
#pragma unroll
    for (int j = 0; j < NTL; ++j) {
        float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (a.bias && nw + 16u * j + 4u * g < a.n) load_row<T, 4>(a.bias, nw + 16u * j + 4u * g, a.n, b);
#pragma unroll
        for (int c = 0; c < 4; ++c) bias[4 * j + c] = b[c];
    }
#pragma unroll 1
    for (int i = 0; i < MT; ++i) {
        const uint32_t m = m0 + wm * TWM + 16u * i + r;
        T *to = reinterpret_cast<T *>(a.out) + (uint64_t)m * a.n;
        float v[NTL * 4];
        auto take = [&](auto row) {
#pragma unroll
            for (int c = 0; c < NTL * 4; ++c) v[c] = acc[decltype(row)::value][c / 4][c % 4] + bias[c];
        };
        switch (i) {
        case 0: take(std::integral_constant<int, 0>()); break;
        case 1: take(std::integral_constant<int, 1>()); break;
        case 2: take(std::integral_constant<int, 2>()); break;
        case 3: take(std::integral_constant<int, 3>()); break;
        case 4: take(std::integral_constant<int, (MT > 4 ? 4 : 0)>()); break;
        case 5: take(std::integral_constant<int, (MT > 4 ? 5 : 0)>()); break;
        case 6: take(std::integral_constant<int, (MT > 4 ? 6 : 0)>()); break;
        default: take(std::integral_constant<int, (MT > 4 ? 7 : 0)>()); break;
        }
        activate(a.act, a.leaky, v);
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < NTL; ++j) {
                const uint32_t col = nw + 16u * j + 4u * g;
                const float w[4] = {v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]};
                if (m < a.m && col < a.n) store_row<T, 4>(to, col, a.n, w);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NTL; j += 2) {
                typedef T T2 __attribute__((ext_vector_type(2)));
                typedef T T8 __attribute__((ext_vector_type(8)));
                u32x4 w;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t lo = __builtin_bit_cast(uint32_t, T2{(T)v[4 * j + 2 * h], (T)v[4 * j + 2 * h + 1]});
                    const uint32_t hi = __builtin_bit_cast(uint32_t, T2{(T)v[4 * j + 4 + 2 * h], (T)v[4 * j + 4 + 2 * h + 1]});
                    const auto both = __builtin_amdgcn_permlane16_swap(lo, hi, false, false);
                    w[h] = both[0];
                    w[2 + h] = both[1];
                }
                const uint32_t col = nw + 16u * (j + (g & 1u)) + 8u * (g >> 1);
                if (m >= a.m || col >= a.n) continue;
                if (col + 8u <= a.n) {
                    *reinterpret_cast<typename Unaligned<T, 8>::type *>(to + col) = __builtin_bit_cast(T8, w);
                } else {
                    const T8 part = __builtin_bit_cast(T8, w);
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        if (col + c < a.n) to[col + c] = part[c];
                }
            }
        }
    }
}

}  // namespace skl

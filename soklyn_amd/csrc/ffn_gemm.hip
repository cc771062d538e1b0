// ffn_gemm.hip — launchers of the products in ffn.h on the direct-to-LDS and K-splitting kernels.
//
//   Pair     out = act(A Wg + bg) * (A Wu + bu)     a tile of both matrices beside each other: A is read once
//   Ungate   s = A B^T, dg = s u act'(a), du = s act(a)     s stays in registers
//   Project  h = scale x + drop(act(A W + b))
//   Chain    dx = A B^T + a2 b2^T                   one k loop over both parts, one store
//
// fp16, 16384 rows (2 M N K of one or two products; HBM as 5.1 TB/s):
//   Pair 2048 -> 4096, a and u kept      466 us: 1.18 PF/s, the library's 8192^3 product 1.14-1.2
//   Chain 2 x 4096 -> 2048               428 us: 1.28 PF/s
//   Project 4096 -> 2048, fp32 stream    260 us: 1.06 PF/s
//   Ungate 2048 -> 4096                  393 us: 0.70 PF/s and 2.9 TB/s; the k loops alone 176, the epilogues'
//     6 tensors alone 226.  All workgroups of a round load, multiply and store together, so the two add up.
#include "ffn.h"
#include "ffn_epi.h"
#include "gemm_dma.h"
#include "gemm_wave.h"

namespace skl {

static bool on4(const void *p, size_t esz) { return (reinterpret_cast<uintptr_t>(p) & (4 * esz - 1)) == 0; }
static bool on16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The epilogue's tensors by groups of `group` columns: rows and bases on whole groups.
static bool rows_on(const ProductLaunch &p, uint32_t group) {
    const size_t t = p.g.dtype == 1 ? 2 : 4, r = p.stream_dtype == 1 ? 2 : 4;
    auto ok = [&](const void *q, size_t esz) { return group == 8 ? on16(q) : on4(q, esz); };
    switch (p.kind) {
    case Product::Pair:
        return p.pair.ldc % group == 0 && ok(p.pair.bias, t) && ok(p.pair.bias2, t) && ok(p.pair.out, t) && ok(p.pair.a, t) &&
               ok(p.pair.u, t);
    case Product::Ungate:
        return p.ungate.ldc % group == 0 && ok(p.ungate.a, t) && ok(p.ungate.u, t) && ok(p.ungate.d_gate, 4) &&
               ok(p.ungate.d_up, 4) && ok(p.ungate.d_gate_h, 2) && ok(p.ungate.d_up_h, 2);
    case Product::Project:
        return p.project.ldc % group == 0 && ok(p.project.bias, t) && ok(p.project.x, r) && ok(p.project.h, r) &&
               ok(p.project.preact, t);
    case Product::Chain: return p.chain.ldc % group == 0 && ok(p.chain.out, 4);
    }
    return false;
}

bool product_rows4(const ProductLaunch &p) { return rows_on(p, 4); }

GemmLaunch planned_gemm(const ProductLaunch &p) {
    GemmLaunch g = p.g;
    auto both = [](const void *x, const void *y) {
        return reinterpret_cast<const void *>(reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y));
    };
    if (p.kind == Product::Pair) {
        g.B = both(g.B, p.pair.b2);
        g.N *= 2;
    }
    if (p.kind == Product::Chain) {
        g.A = both(g.A, p.chain.a2);
        g.B = both(g.B, p.chain.b2);
        g.K *= 2;
    }
    return g;
}

bool product_registers(const ProductLaunch &p) { return !wave_dword_rows(planned_gemm(p)); }

// ---- direct-to-LDS ---------------------------------------------------------------------
template <class Epi, bool BK, int NW, bool EDGE, int BT, bool RAG>
static hipError_t run_dma(const ProductLaunch &p, const typename Epi::Params &e, bool whole, hipStream_t s) {
    const GemmLaunch &g = p.g;
    constexpr uint32_t TN = EpiPair<Epi>::value ? BT / 2 : BT;
    GemmShape sh{};
    sh.M = g.M;
    sh.N = g.N;
    sh.K = g.K;
    sh.lda = g.lda;
    sh.ldb = g.ldb;
    sh.k_per_split = (g.K + 127) / 128 * 128;
    sh.tiles_m = (g.M + BT - 1) / BT;
    sh.tiles_n = (g.N + TN - 1) / TN;
    sh.mv = g.mv;
    sh.nv = g.nv;
    sh.whole = whole;
    launch_timed(g, gemm_dma_kernel<Epi, true, BK, NW, EDGE, 16, BT, RAG>, dim3(sh.tiles_m * sh.tiles_n), dim3(64 * NW), s,
                 sh, reinterpret_cast<const half_t *>(g.A), reinterpret_cast<const half_t *>(g.B), e);
    return hipGetLastError();
}

// 256x256 tiles on 8 waves, but for the plain store of a chain, which takes one wave per SIMD where
// the tiles are whole; 128x128 on 4; both also over padded copies (mv, nv the real output), 128x128
// over operands as stored.  The epilogues of the others want the threads of 8 waves (4 waves of 128x128:
// 2-4% slower), and 128x128 tiles, two workgroups to a CU, lose more in the k loop than their epilogues
// gain beside it (Pair 545 us, Project 308, Ungate 442).
template <class Epi, bool BK>
static hipError_t dma(const ProductLaunch &p, const typename Epi::Params &e, hipStream_t s) {
    const GemmLaunch &g = p.g;
    const bool whole = rows_on(p, EpiPair<Epi>::value ? 8 : 4);
    if (g.rag) return run_dma<Epi, BK, 4, true, 128, true>(p, e, whole, s);
    const bool edge = !whole || g.mv != g.M || g.nv != g.N;
    if (g.tile == 128)
        return edge ? run_dma<Epi, BK, 4, true, 128, false>(p, e, whole, s)
                    : run_dma<Epi, BK, 4, false, 128, false>(p, e, whole, s);
    if (edge) return run_dma<Epi, BK, 8, true, 256, false>(p, e, whole, s);
    if constexpr (EpiChain<Epi>::value) return run_dma<Epi, BK, 4, false, 256, false>(p, e, whole, s);
    else return run_dma<Epi, BK, 8, false, 256, false>(p, e, whole, s);
}

static hipError_t launch_dma(const ProductLaunch &p, hipStream_t s) {
    const GemmLaunch &g = p.g;
    if (g.dtype != 1 || !g.M || !g.N || !g.K) return hipErrorInvalidValue;
    const GemmLaunch all = planned_gemm(p);
    if (g.rag) {
        if (g.K % 8 || !gemm_dma_rag_ok(all)) return hipErrorInvalidValue;
    } else {
        const uint32_t t = g.tile == 128 ? 128 : 256, tn = p.kind == Product::Pair ? t / 2 : t;
        if (g.M % t || g.N % tn || g.K % (p.kind == Product::Chain ? 64 : 128) || g.lda % 8 || g.ldb % 8 || !on16(all.A) ||
            !on16(all.B))
            return hipErrorInvalidValue;
    }
    switch (p.kind) {
    case Product::Pair: return dma<EpiPairK<half_t>, false>(p, p.pair, s);
    case Product::Ungate: return dma<EpiUngateK<half_t>, true>(p, p.ungate, s);
    case Product::Project:
        return p.stream_dtype == 1 ? dma<EpiProjectK<half_t, half_t>, false>(p, p.project, s)
                                   : dma<EpiProjectK<half_t, float>, false>(p, p.project, s);
    case Product::Chain: return dma<EpiChainK, true>(p, p.chain, s);
    }
    return hipErrorInvalidValue;
}

// ---- K-splitting -------------------------------------------------------------------------
// A pair's tile is 16x16, 32x16 or 64x32 of each matrix (the LDS and accumulators of 16x32, 32x32
// and 64x64 of one), the others' 16, 32 or 64 squared.
static uint32_t wave_rows(const ProductLaunch &p) { return p.g.tile; }
static uint32_t wave_cols(const ProductLaunch &p) {
    return p.kind != Product::Pair ? p.g.tile : p.g.tile == 16 ? 16 : p.g.tile / 2;
}
static uint64_t wave_tiles(const ProductLaunch &p) {
    const uint32_t r = wave_rows(p), c = wave_cols(p);
    return (uint64_t)((p.g.M + r - 1) / r) * ((p.g.N + c - 1) / c);
}
// (16 waves of a pair's 16x16 tiles would not leave the registers for the sum over them)
static uint32_t wave_waves(const ProductLaunch &p) {
    return p.kind == Product::Pair && p.g.tile == 16 ? 8 : p.g.waves ? p.g.waves : gemm_wave_waves(planned_gemm(p), p.g.tile);
}
uint64_t product_threads(const ProductLaunch &p) { return wave_tiles(p) * 64 * wave_waves(p); }

template <typename T, class Epi, bool BK, bool REG, int MB, int W, int S, int WPE>
static hipError_t run_wave_t(const ProductLaunch &p, const typename Epi::Params &e, hipStream_t s) {
    constexpr int NB = EpiPair<Epi>::value && MB > 1 ? MB / 2 : MB;
    const GemmLaunch &g = p.g;
    GemmShape sh{};
    sh.M = g.M;
    sh.N = g.N;
    sh.K = g.K;
    sh.lda = g.lda;
    sh.ldb = g.ldb;
    sh.tiles_m = (g.M + 16 * MB - 1) / (16 * MB);
    sh.tiles_n = (g.N + 16 * NB - 1) / (16 * NB);
    sh.k_per_split = gemm_wave_slice(g.K, 1);
    sh.nv = rows_on(p, 4);
    launch_timed(g, gemm_wave_kernel<T, Epi, true, BK, REG, MB, NB, W, S, WPE>, dim3(sh.tiles_m * sh.tiles_n), dim3(64 * W),
                 s, sh, reinterpret_cast<const T *>(g.A), reinterpret_cast<const T *>(g.B), e);
    return hipGetLastError();
}

template <typename T, class Epi, bool BK>
static hipError_t wave(const ProductLaunch &p, const typename Epi::Params &e, hipStream_t s) {
    constexpr bool PAIR = EpiPair<Epi>::value;
    const uint32_t code = p.g.tile * 32 + wave_waves(p);
    if constexpr (sizeof(T) == 2) {
        if (product_registers(p)) {
            switch (code) {
            case 16 * 32 + 8: if constexpr (PAIR) return run_wave_t<T, Epi, BK, true, 1, 8, 1, 2>(p, e, s); break;
            case 16 * 32 + 16: if constexpr (!PAIR) return run_wave_t<T, Epi, BK, true, 1, 16, 1, 4>(p, e, s); break;
            // (a chain's two sets of addresses pass the registers of four waves to a SIMD)
            case 32 * 32 + 8: return run_wave_t<T, Epi, BK, true, 2, 8, 1, EpiChain<Epi>::value ? 2 : 4>(p, e, s);
            case 64 * 32 + 4: return run_wave_t<T, Epi, BK, true, 4, 4, 1, 2>(p, e, s);
            }
            return hipErrorInvalidValue;
        }
        switch (code) {
        case 16 * 32 + 8: if constexpr (PAIR) return run_wave_t<T, Epi, BK, false, 1, 8, 2, 2>(p, e, s); break;
        case 16 * 32 + 16: if constexpr (!PAIR) return run_wave_t<T, Epi, BK, false, 1, 16, 2, 4>(p, e, s); break;
        case 32 * 32 + 4: return run_wave_t<T, Epi, BK, false, 2, 4, 2, 2>(p, e, s);
        case 64 * 32 + 2: return run_wave_t<T, Epi, BK, false, 4, 2, 1, 2>(p, e, s);
        case 64 * 32 + 4: return run_wave_t<T, Epi, BK, false, 4, 4, 1, 2>(p, e, s);
        }
    } else {
        switch (code) {
        case 16 * 32 + 8: if constexpr (PAIR) return run_wave_t<T, Epi, BK, false, 1, 8, 2, 2>(p, e, s); break;
        case 16 * 32 + 16: if constexpr (!PAIR) return run_wave_t<T, Epi, BK, false, 1, 16, 2, 4>(p, e, s); break;
        case 32 * 32 + 8: return run_wave_t<T, Epi, BK, false, 2, 8, 1, 4>(p, e, s);
        case 64 * 32 + 8: return run_wave_t<T, Epi, BK, false, 4, 8, 1, 2>(p, e, s);
        case 64 * 32 + 4: return run_wave_t<T, Epi, BK, false, 4, 4, 1, 2>(p, e, s);
        case 64 * 32 + 2: return run_wave_t<T, Epi, BK, false, 4, 2, 1, 2>(p, e, s);
        case 64 * 32 + 1: return run_wave_t<T, Epi, BK, false, 4, 1, 1, 2>(p, e, s);
        }
    }
    return hipErrorInvalidValue;
}

template <typename T> static hipError_t launch_wave(const ProductLaunch &p, hipStream_t s) {
    switch (p.kind) {
    case Product::Pair: return wave<T, EpiPairK<T>, false>(p, p.pair, s);
    case Product::Ungate: return wave<T, EpiUngateK<T>, true>(p, p.ungate, s);
    case Product::Project:
        if constexpr (sizeof(T) == 2)
            if (p.stream_dtype == 1) return wave<T, EpiProjectK<T, half_t>, false>(p, p.project, s);
        return wave<T, EpiProjectK<T, float>, false>(p, p.project, s);
    case Product::Chain: return wave<T, EpiChainK, true>(p, p.chain, s);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_product(const ProductLaunch &p, hipStream_t s) {
    if (p.dma) return launch_dma(p, s);
    if (!p.g.M || !p.g.N || !p.g.K || product_threads(p) > 0xffffffffull) return hipErrorInvalidValue;
    return p.g.dtype == 1 ? launch_wave<half_t>(p, s) : launch_wave<float>(p, s);
}

}  // namespace skl

// ffn.h — launchers of the gated feed-forward block, the projection into the residual stream and
// dropout (ffn_gemm.hip, ffn.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.h"

namespace skl {

// Dropout without a stored mask: an element stays where dropout_bits of its column, row and seed
// (seed + 7 row, as the blocks draw theirs) is at least keep_min, times `scale` = 1 / (1 - p).
struct DropArgs {
    uint32_t on, seed, keep_min;
    float scale;
};
inline DropArgs drop_args(bool on, float p, uint32_t seed) {
    DropArgs d{};
    if (!on || !(p > 0.0f)) return d;
    d.on = 1;
    d.seed = seed;
    d.keep_min = (uint32_t)dropout_keep_min(p);   // p < 1: below 2^32
    d.scale = 1.0f / (1.0f - p);
    return d;
}
__device__ __forceinline__ float drop_factor(const DropArgs &d, uint32_t colmul, uint32_t rowkey) {
    return dropout_bits(colmul, rowkey) >= d.keep_min ? d.scale : 0.0f;
}
__device__ __forceinline__ uint32_t drop_rowkey(const DropArgs &d, uint32_t row) {
    return dropout_rowkey(row, d.seed + row * 7u);
}

// ---- what the products do with an output element ----------------------------------------
// out = act(a) * u of a = x . Wg + bg and u = x . Wu + bu; a and u, rounded, to their caches.
struct PairEpi {
    const void *b2;               // Wu (T)
    const void *bias, *bias2;     // T [n] or null
    void *out, *a, *u;            // T [m x ldc]; a, u may be null
    uint32_t act, ldc;
    float leaky, pad;
};
// From the sum s: the gradients of a and u.
struct UngateEpi {
    const void *a, *u;            // T [m x ldc]
    float *d_gate, *d_up;
    half_t *d_gate_h, *d_up_h;    // fp16 blocks
    uint32_t act, ldc;
    float leaky, pad;
};
// h = scale * x + dropout(act(z)), z = in . W + b; z, rounded, to preact.
struct ProjectEpi {
    const void *bias;             // T [n] or null
    const void *x;                // R [m x ldc] or null
    void *h;                      // R [m x ldc]; may be x
    void *preact;                 // T [m x ldc] or null
    uint32_t act, ldc;
    float leaky, scale;
    DropArgs drop;
};
// dx = A . B^T + a2 . b2^T (fp32)
struct ChainEpi {
    float *out;
    const void *a2, *b2;          // T, pitches as A and B
    uint32_t ldc, pad;
};

enum class Product { Pair, Ungate, Project, Chain };

// One product.  g: sizes, operands, pitches, the kernel (dma: direct-to-LDS with its tile, rag and
// mv, nv; else the K-splitting kernel on g.tile) and the timing events.  g.N is the output's
// columns, for a Pair those of each matrix; g.K is for a Chain the length of each part.
struct ProductLaunch {
    GemmLaunch g;
    Product kind;
    bool dma;
    uint32_t stream_dtype;        // Project: type of x and h
    PairEpi pair;
    UngateEpi ungate;
    ProjectEpi project;
    ChainEpi chain;
};
hipError_t launch_product(const ProductLaunch &p, hipStream_t s);
// The GEMM as which a product is planned and its kernel's form chosen: of twice the columns (Pair) or
// twice the k (Chain).  Its addresses stand for the alignment of all operands, the second ones too.
GemmLaunch planned_gemm(const ProductLaunch &p);
// The K-splitting kernel takes the operands through registers: rows off 4-byte boundaries.
bool product_registers(const ProductLaunch &p);
// The kernels for few rows of a Pair or Project (ffn_rows.hip), which want product_rows_bytes of
// workspace: whether sizes are theirs, and a product with its alignments.
hipError_t launch_product_rows(const ProductLaunch &p, void *work, hipStream_t s);
bool product_rows_size(uint32_t dtype, uint32_t M, uint32_t N, uint32_t K, uint32_t matrices);
bool product_rows_ok(const ProductLaunch &p);
size_t product_rows_bytes(uint32_t M, uint32_t N, uint32_t matrices);
// Every tensor of the epilogue starts its rows on 4 elements.
bool product_rows4(const ProductLaunch &p);
// Threads of the K-splitting kernel's launch.
uint64_t product_threads(const ProductLaunch &p);

// ---- element-wise kernels ----------------------------------------------------------------
// The gradients of a and u from s, the gradient of act(a) * u, over n elements.
struct UngateArgs {
    uint64_t n;
    const float *s;
    UngateEpi e;
};
hipError_t launch_ungate(const UngateArgs &a, uint32_t dtype, hipStream_t s);

// d = dropout's factor * dh * act'(preact), its fp16 copy, and dx = scale * dh.
struct UnprojectArgs {
    uint32_t rows, cols;
    const float *dh;
    const void *preact;           // T
    float *d_prenorm, *dx;        // dx may be null, or dh
    half_t *d_prenorm_h;
    uint32_t act;
    float leaky, scale;
    DropArgs drop;
};
hipError_t launch_unproject(const UnprojectArgs &a, uint32_t dtype, hipStream_t s);

struct DropoutArgs {
    uint32_t rows, cols;
    const void *in;               // T
    void *out;                    // T; may be in
    DropArgs drop;
};
hipError_t launch_dropout(const DropoutArgs &a, uint32_t dtype, hipStream_t s);

}  // namespace skl

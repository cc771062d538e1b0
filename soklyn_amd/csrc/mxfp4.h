// mxfp4.h — launchers of the 4-bit microscaled float kernels (mxfp4.hip).
//
// A matrix of n vectors of k elements is held as codes [n][kp / 2] and scales [n][kp / 32], kp = k
// rounded up to 128: element i of a vector is the low (i even) or high half of byte i / 2, an
// e2m1 float (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), times the
// scale 2^(byte - 127) of its block of 32; byte 255 makes the block NaN.  Elements past k are 0.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "launch.h"

namespace skl {

inline __host__ __device__ uint32_t mx_pad(uint32_t k) { return (k + 127u) / 128u * 128u; }
inline __host__ __device__ uint32_t mx_ceil(uint32_t v, uint32_t by) { return v / by + (v % by != 0); }

// Columns of a workgroup of the casts down the columns, which takes 128 rows of them, 256 threads.
inline constexpr uint32_t mx_down_cols(size_t element) { return (uint32_t)(256 / element); }
// A launch has less than 2^32 threads (along the rows workgroups loop).
inline bool mx_cast_fits(uint32_t n, uint32_t k, bool down, size_t element) {
    return !down || (uint64_t)mx_ceil(n, mx_down_cols(element)) * (mx_pad(k) / 128u) * 256u <= 0xffffffffu;
}

struct MxCastArgs {
    uint32_t n, k;          // vectors and their length
    void *values;           // T
    uint8_t *codes, *scales;
};
hipError_t launch_mx_quantise(const MxCastArgs &a, uint32_t dtype, bool down, hipStream_t s);
hipError_t launch_mx_dequantise(const MxCastArgs &a, uint32_t dtype, bool down, hipStream_t s);

constexpr uint32_t kMxInputs = 1u << 24;   // a tile's codes, 256 vectors, are within 2^32 bytes

struct MxForwardArgs {
    uint32_t m, n, k;
    const void *x;                      // T [m x k]
    const uint8_t *w_codes, *w_scales;  // n vectors of k
    const void *bias;                   // T [n] or null
    uint32_t act;
    float leaky;
    void *out;                          // T [m x n]
    void *work;                         // mx_work(k, n, m).bytes
};

// The tile edge of the product, 0: the kernel for few rows, which needs no workspace.  64 x 64 tiles,
// whose waves split the k axis, while the GPU holds them all at once (256 rows by 4096 x 4096: 15.9 us,
// 18.8 on 128 x 128; 512 rows: 27.1 and 20.3), 256 x 256 once they leave few CUs idle (3000 rows:
// 47.2 us, 50.6 on 128 x 128; 2048 rows: 40.7 and 36.4; 8192 rows: 95.3 and 110.6), 128 x 128 between.
// 16 rows: 9.6 us without staging, 14.6 with; 32 rows: 12.9 and 14.8.
inline uint32_t mx_tile(uint32_t m, uint32_t n) {
    auto tiles = [&](uint32_t t) { return (uint64_t)mx_ceil(m, t) * mx_ceil(n, t); };
    return m <= 32 ? 0 : tiles(64) <= 256 ? 64 : tiles(256) >= 160 ? 256 : 128;
}

// The workspace of the tiled product: x's codes, then both scales in the product's order.
struct MxWork {
    size_t mp, np, k2;   // padded: rows, outputs, inputs
    size_t codes, xs, ws, bytes;
};
inline MxWork mx_work(uint32_t k, uint32_t n, uint32_t m) {
    MxWork w{};
    const uint32_t t = mx_tile(m, n);
    if (t == 0) return w;
    w.mp = (size_t)mx_ceil(m, t) * t;
    w.np = (size_t)mx_ceil(n, t) * t;
    w.k2 = (size_t)mx_ceil(k, 256) * 256;
    w.codes = w.mp * (w.k2 / 2);
    w.xs = w.mp * (w.k2 / 32);
    w.ws = w.np * (w.k2 / 32);
    w.bytes = w.codes + w.xs + w.ws;
    return w;
}

// A launch has less than 2^32 threads.  Staging: 256 for 64 rows by 128 inputs, and for 64 outputs by 512.
inline uint64_t mx_stage_x(const MxWork &w) { return w.mp / 64 * (w.k2 / 128); }
inline uint64_t mx_stage_groups(const MxWork &w) { return mx_stage_x(w) + w.np / 64 * ((w.k2 + 511) / 512); }
inline bool mx_fits(uint32_t k, uint32_t n, uint32_t m) {
    const uint32_t t = mx_tile(m, n);
    if (t == 0) return (uint64_t)mx_ceil(n, 16) * 512 <= 0xffffffffu;
    return mx_stage_groups(mx_work(k, n, m)) * 256 <= 0xffffffffu &&
           (uint64_t)mx_ceil(m, t) * mx_ceil(n, t) * 512 <= 0xffffffffu;
}
hipError_t launch_mx_forward(const MxForwardArgs &a, uint32_t dtype, hipStream_t s);

}  // namespace skl

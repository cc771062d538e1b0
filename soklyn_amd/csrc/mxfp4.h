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
    auto tiles = [&](uint32_t t) { return (uint64_t)((m + t - 1) / t) * ((n + t - 1) / t); };
    return m <= 32 ? 0 : tiles(64) <= 256 ? 64 : tiles(256) >= 160 ? 256 : 128;
}

// The workspace of the tiled product: x's codes, then both scales in the product's order.
struct MxWork {
    uint32_t mp, np, k2;
    size_t codes, xs, ws, bytes;
};
inline MxWork mx_work(uint32_t k, uint32_t n, uint32_t m) {
    MxWork w{};
    const uint32_t t = mx_tile(m, n);
    if (t == 0) return w;
    w.mp = (m + t - 1) / t * t;
    w.np = (n + t - 1) / t * t;
    w.k2 = (k + 255u) / 256u * 256u;
    w.codes = (size_t)w.mp * (w.k2 / 2);
    w.xs = (size_t)w.mp * (w.k2 / 32);
    w.ws = (size_t)w.np * (w.k2 / 32);
    w.bytes = w.codes + w.xs + w.ws;
    return w;
}
hipError_t launch_mx_forward(const MxForwardArgs &a, uint32_t dtype, hipStream_t s);

}  // namespace skl

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

// The tile edge of the product, 0: the kernel for few rows, which needs no workspace.
inline uint32_t mx_tile(uint32_t m, uint32_t n) {
    const uint64_t t256 = (uint64_t)((m + 255) / 256) * ((n + 255) / 256);
    const uint64_t t128 = (uint64_t)((m + 127) / 128) * ((n + 127) / 128);
    return t256 >= 192 ? 256 : t128 >= 64 ? 128 : 0;
}

// The workspace of the tiled product: x's codes, then both scales in the product's order.
struct MxWork {
    uint32_t mp, np, k2;
    size_t codes, xs, ws, bytes;
};
inline MxWork mx_work(uint32_t k, uint32_t n, uint32_t m) {
    MxWork w{};
    if (mx_tile(m, n) == 0) return w;
    w.mp = (m + 255u) / 256u * 256u;
    w.np = (n + 255u) / 256u * 256u;
    w.k2 = (k + 255u) / 256u * 256u;
    w.codes = (size_t)w.mp * (w.k2 / 2);
    w.xs = (size_t)w.mp * (w.k2 / 32);
    w.ws = (size_t)w.np * (w.k2 / 32);
    w.bytes = w.codes + w.xs + w.ws;
    return w;
}
hipError_t launch_mx_forward(const MxForwardArgs &a, uint32_t dtype, hipStream_t s);

}  // namespace skl

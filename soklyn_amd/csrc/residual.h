// residual.h — launchers of the residual join and its backward (residual.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace skl {

constexpr uint32_t kJoinCols = 8192;   // a row is held in the registers of one workgroup
constexpr int kPlanes = 5;             // column sums: post_w, post_b, pre_w, pre_b, one gate row

struct JoinArgs {
    uint32_t rows, cols, post, pre, gate_act, gate_rows;
    float scale;
    const void *x, *y, *gate, *post_w, *post_b, *pre_w, *pre_b;
    void *h, *n;
    float *stats;   // [4 x rows] or null
};

struct UnjoinArgs {
    uint32_t rows, cols, post, pre, gate_act, gate_rows;
    float scale;
    const void *h, *y, *gate, *post_w, *post_b, *pre_w;
    const float *stats, *dn, *dh;
    float *dx, *dy;
    float *dgate;      // per-row gates
    float *gate_sum;   // one gate row: its column sums
    float *dparam;     // [4 x cols]
    uint32_t planes;   // bit p: column sum p is wanted and not zero
    float *work;       // null: no column sums wanted
};

// The most workgroups of the backward of [rows x cols] (rows > 0), each of which writes a plane of column sums.
inline uint32_t residual_planes(uint32_t rows, uint32_t cols) {
    const uint32_t rpg = cols <= 64 ? 16 : cols <= 512 ? 4 : 1;
    const uint32_t groups = (rows - 1) / rpg + 1, most = cols <= 1024 ? 1280 : cols <= 2048 ? 768 : 256;
    return groups < most ? groups : most;
}

hipError_t launch_join(const JoinArgs &a, uint32_t dtype, uint32_t stream_dtype, hipStream_t s);
hipError_t launch_unjoin(const UnjoinArgs &a, uint32_t dtype, uint32_t stream_dtype, hipStream_t s);

}  // namespace skl

// distill.h — launcher of the distillation error (distill.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_math.h"

namespace skl {

constexpr uint32_t kDistillTop = 1024;   // teacher logits per row: four to six LDS words each

struct DistillArgs {
    uint32_t rows, n, top;
    float tau, alpha;
    const void *logits;         // T [rows x n]
    const int32_t *index;       // [rows x top], outside [0, n): empty
    const float *value;         // [rows x top]
    const int32_t *label;       // [rows] or null, outside [0, n): none
    float *loss;                // [rows] or null
    float *grad, *d_prenorm;    // [rows x n]
    half_t *d_prenorm_h;        // fp16 layers
};

hipError_t launch_distill(const DistillArgs &a, uint32_t dtype, hipStream_t s);

}  // namespace skl

// distill.hip — the error of an output layer that learns from a teacher's top logits.  Per row,
// with z the layer's logits, v_j at class i_j the teacher's (j over the row's held slots), t the
// temperature and y the label:
//
//   q = softmax_j(v / t),  p = softmax(z / t),  p1 = softmax(z)
//   loss = alpha t^2 sum_j q_j (log q_j - log p[i_j]) - (1 - alpha) log p1[y]
//   d loss / d z = alpha t (p - q) + (1 - alpha) (p1 - [y])
//
// the gradient times the loss scale into grad and d_prenorm (and its fp16 copy).  A row without
// held slots has no first term, one without a label no second, and one whose logits are all -inf
// neither; NaN and +inf logits make their row NaN, as in a softmax.
#include "distill.h"
#include "launch.h"
#include "rows.h"

namespace skl {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 2^((v - m) k), m a maximum; m = -inf (no finite value) counts as 0: then -inf gives 0, NaN NaN.
__device__ __forceinline__ float exp2_from(float v, float m, float k) {
    return __builtin_amdgcn_exp2f((v - (m == -INFINITY ? 0.0f : m)) * k);
}

__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}

// Orders a row's LDS accesses among its NT threads; a wave's own are executed in order.
template <int NT> __device__ __forceinline__ void row_sync() {
    if constexpr (NT > 64) {
        __syncthreads();
    } else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// NT threads to a row (64: four rows to a workgroup), E > 0: which hold it in registers, E
// elements each, from one read; E = 0: rows longer than that are read three times (maximum, sums,
// gradient).  LDS per row: the teacher's classes, logits and shares, and a bit for each 2^group
// columns that says whether a slot or the label may be among them, so that the pass over the
// columns looks at the slots only there and every gradient is written once.
template <typename T, int NT, int E> __global__ void __launch_bounds__(NT < 256 ? 256 : NT) distill_kernel(DistillArgs a) {
    constexpr int V = 16 / sizeof(T), W = NT / 64, C = E / V, RPG = NT < 256 ? 256 / NT : 1;
    constexpr uint32_t kMarks = NT < 256 ? 32 : 256;   // words
    typedef typename Unaligned<T, V>::type Vec;
    extern __shared__ uint32_t lds[];
    __shared__ float red[4][W];
    const uint32_t tid = threadIdx.x % NT, lane = threadIdx.x & 63u, n = a.n, top = a.top;
    uint32_t *marks = lds + (threadIdx.x / NT) * (kMarks + 3 * top);
    int32_t *at = reinterpret_cast<int32_t *>(marks + kMarks);
    float *value = reinterpret_cast<float *>(at + top), *q = value + top;
    const float k_soft = kLog2e / a.tau;
    uint32_t group = 0;
    while ((n - 1) >> group >= kMarks * 32u) ++group;

    for (uint32_t row = blockIdx.x * RPG + threadIdx.x / NT; row < a.rows; row += gridDim.x * RPG) {
        const T *z = reinterpret_cast<const T *>(a.logits) + (uint64_t)row * n;
        Vec held[E > 0 ? C : 1];
        if constexpr (E > 0) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const uint32_t col = (c * NT + tid) * V;
                if (col + V <= n) {
                    held[c] = *reinterpret_cast<const Vec *>(z + col);
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) held[c][e] = col + e < n ? z[col + e] : (T)-INFINITY;
                }
            }
        }
        // every column's values by f(column, values)
        auto each = [&](auto f) {
            if constexpr (E > 0) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    float v[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] = (float)held[c][e];
                    f((c * NT + tid) * V, v);
                }
            } else {
                for (uint32_t col = tid * V; col < n; col += NT * V) {
                    float v[V];
                    load_row<T, V>(z, col, n, v, -INFINITY);
                    f(col, v);
                }
            }
        };

        // the teacher's slots and the label
        for (uint32_t j = tid; j < kMarks; j += NT) marks[j] = 0;
        for (uint32_t j = tid; j < top; j += NT) {
            const int32_t i = a.index[(uint64_t)row * top + j];
            const bool in = (uint32_t)i < n;
            at[j] = in ? i : -1;
            value[j] = in ? a.value[(uint64_t)row * top + j] : -INFINITY;
        }
        const int32_t y = a.label ? a.label[row] : -1;
        row_sync<NT>();
        // each wave for itself, in one order: the largest logit, then the sum
        float t_max = -INFINITY, t_sum = 0.0f;
        for (uint32_t j = lane; j < top; j += 64) t_max = fmaxf(t_max, value[j]);
        t_max = lanes_max(t_max);
        for (uint32_t j = lane; j < top; j += 64) t_sum += at[j] >= 0 ? exp2_from(value[j], t_max, k_soft) : 0.0f;
        t_sum = lanes_sum(t_sum);
        const bool taught = a.alpha > 0.0f && t_sum != 0.0f;   // NaN: taught, and NaN
        for (uint32_t j = tid; j < top; j += NT) {
            q[j] = taught && at[j] >= 0 ? exp2_from(value[j], t_max, k_soft) / t_sum : 0.0f;
            if (at[j] >= 0) atomicOr(&marks[(uint32_t)at[j] >> group >> 5], 1u << ((uint32_t)at[j] >> group & 31u));
        }
        const bool labelled = (uint32_t)y < n;
        if (tid == 0 && labelled) atomicOr(&marks[(uint32_t)y >> group >> 5], 1u << ((uint32_t)y >> group & 31u));

        // the layer's maximum and sums
        float m = -INFINITY;
        each([&](uint32_t, const float (&v)[V]) {
#pragma unroll
            for (int e = 0; e < V; ++e) m = fmaxf(m, v[e]);
        });
        m = lanes_max(m);
        if constexpr (NT > 64) {
            if (lane == 0) red[0][tid >> 6] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < W; ++w) m = fmaxf(m, red[0][w]);
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float s_soft = 0.0f, s_hard = 0.0f;
        if (taught)
            each([&](uint32_t, const float (&v)[V]) {
#pragma unroll
                for (int e = 0; e < V; ++e) s_soft += __builtin_amdgcn_exp2f((v[e] - base) * k_soft);
            });
        if (labelled)
            each([&](uint32_t, const float (&v)[V]) {
#pragma unroll
                for (int e = 0; e < V; ++e) s_hard += __builtin_amdgcn_exp2f((v[e] - base) * kLog2e);
            });
        s_soft = row_sum<NT>(s_soft, red[1]);
        s_hard = row_sum<NT>(s_hard, red[2]);
        // a sum of 0: all logits -inf
        const bool soft = taught && s_soft != 0.0f, hard = labelled && s_hard != 0.0f;
        const float g_soft = soft ? kLossScale * a.alpha * a.tau : 0.0f;
        const float g_hard = hard ? kLossScale * (1.0f - a.alpha) : 0.0f;
        const float c_soft = soft ? g_soft / s_soft : 0.0f, c_hard = hard ? g_hard / s_hard : 0.0f;

        const uint64_t row_at = (uint64_t)row * n;
        row_sync<NT>();   // q and marks
        each([&](uint32_t col, const float (&v)[V]) {
            if (E > 0 && col >= n) return;
            float g[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                g[e] = soft ? c_soft * __builtin_amdgcn_exp2f((v[e] - base) * k_soft) : 0.0f;
                if (hard) g[e] += c_hard * __builtin_amdgcn_exp2f((v[e] - base) * kLog2e);
            }
            uint32_t marked = 0;   // a group holds a whole vector, or (group < 3) several bits cover one
            for (uint32_t b = col >> group; b <= min(col + V - 1, n - 1) >> group; ++b) marked |= marks[b >> 5] >> (b & 31u) & 1u;
            if (marked) {
                if (soft)
                    for (uint32_t j = 0; j < top; ++j) {
                        const uint32_t off = (uint32_t)at[j] - col;   // an empty slot's is past V
#pragma unroll
                        for (int e = 0; e < V; ++e) g[e] -= off == (uint32_t)e ? g_soft * q[j] : 0.0f;
                    }
#pragma unroll
                for (int e = 0; e < V; ++e) g[e] -= (uint32_t)y == col + e ? g_hard : 0.0f;
            }
            store_row<float, V>(a.grad + row_at, col, n, g);
            store_row<float, V>(a.d_prenorm + row_at, col, n, g);
            if constexpr (sizeof(T) == 2) store_row<half_t, V>(a.d_prenorm_h + row_at, col, n, g);
        });

        float l = 0.0f;
        if (a.loss && soft) {
            const float log_p = __builtin_amdgcn_logf(s_soft), log_q = __builtin_amdgcn_logf(t_sum);
            for (uint32_t j = tid; j < top; j += NT)
                if (at[j] >= 0 && q[j] != 0.0f)
                    l += q[j] * (((value[j] - t_max) * k_soft - log_q) - ((to_f32(z[at[j]]) - base) * k_soft - log_p));
        }
        if (a.loss) l = row_sum<NT>(l, red[3]);
        if (a.loss && tid == 0) {
            l *= a.alpha * a.tau * a.tau * kLn2;
            if (hard) l -= (1.0f - a.alpha) * kLn2 * ((to_f32(z[y]) - base) * kLog2e - __builtin_amdgcn_logf(s_hard));
            a.loss[row] = l;
        }
        row_sync<NT>();   // the next row's slots
    }
}

template <typename T, int NT, int E> hipError_t distill_t(const DistillArgs &a, hipStream_t s) {
    constexpr uint32_t rpg = NT < 256 ? 256 / NT : 1, marks = NT < 256 ? 32 : 256;
    const uint32_t groups = (a.rows + rpg - 1) / rpg;
    hipLaunchKernelGGL((distill_kernel<T, NT, E>), dim3(groups < (1u << 20) ? groups : 1u << 20),
                       dim3(NT < 256 ? 256 : NT), rpg * (marks + 3 * a.top) * 4, s, a);
    return hipGetLastError();
}

template <typename T> hipError_t distill_n(const DistillArgs &a, hipStream_t s) {
    if (a.n <= 512) return distill_t<T, 64, 8>(a, s);
    if (a.n <= 1024) return distill_t<T, 64, 16>(a, s);
    if (a.n <= 2048) return distill_t<T, 256, 8>(a, s);
    if (a.n <= 16384) return distill_t<T, 256, 0>(a, s);
    return distill_t<T, 1024, 0>(a, s);
}

}  // namespace

hipError_t launch_distill(const DistillArgs &a, uint32_t dtype, hipStream_t s) {
    return dtype ? distill_n<half_t>(a, s) : distill_n<float>(a, s);
}

}  // namespace skl

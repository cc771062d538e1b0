// residual.hip — the join between two blocks of a residual network, forward and backward:
//
//   u = post(y)                    the norm behind the block (none, RMS, Layer)
//   h = scale x + act(gate) u      the residual stream, rounded to its type
//   n = pre(h)                     the norm before the next block, of h as stored
//
// A row is held in registers, 8 or 16 elements a thread, from its loads to its stores, so each
// tensor crosses HBM once; the norms' sums are two-pass (mean, then squared deviations).
#include "launch.h"
#include "residual.h"
#include "rows.h"

namespace skl {

constexpr float kNormEps = 1e-6f;   // the blocks' own norms add the same

namespace {

__device__ __forceinline__ float gate_value(uint32_t act, float g) {
    if (act == 1) return 1.0f / (1.0f + expf(-g));
    if (act == 4) return tanhf(g);
    return g;
}
// The gate's slope from its value a.
__device__ __forceinline__ float gate_slope(uint32_t act, float a) {
    if (act == 1) return a * (1.0f - a);
    if (act == 4) return 1.0f - a * a;
    return 1.0f;
}

// Mean and reciprocal deviation of a row's values v (zero past its end).
template <int NT, int E, int V>
__device__ __forceinline__ void row_stats(const float (&v)[E], uint32_t tid, uint32_t cols, uint32_t norm, float *slots,
                                          float &mean, float &rstd) {
    mean = 0.0f;
    rstd = 1.0f;
    if (norm == 0) return;
    const float inv = 1.0f / (float)cols;
    if (norm == 2) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += v[e];
        mean = row_sum<NT>(s, slots) * inv;
    }
    float q = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const uint32_t col = ((uint32_t)(e / V) * NT + tid) * V + e % V;
        const float d = col < cols ? v[e] - mean : 0.0f;
        q += d * d;
    }
    rstd = 1.0f / sqrtf(row_sum<NT>(q, slots + NT / 64) * inv + kNormEps);
}

// One row per NT threads (four rows per workgroup where a wave is enough for one).
template <typename T, typename R, int NT, int E>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) join_kernel(JoinArgs a) {
    constexpr int V = 16 / sizeof(T), C = E / V;
    constexpr int RPG = NT < 256 ? 256 / NT : 1;
    __shared__ float slots[4 * (NT / 64)];
    const uint32_t tid = threadIdx.x % NT;
    const uint32_t cols = a.cols;
    auto chunk = [&](int c) { return ((uint32_t)c * NT + tid) * V; };
    auto part = [&](float (&v)[E], int c) -> float (&)[V] { return *reinterpret_cast<float (*)[V]>(&v[c * V]); };
    for (uint32_t row = blockIdx.x * RPG + threadIdx.x / NT; row < a.rows; row += gridDim.x * RPG) {
    const uint64_t at = (uint64_t)row * cols;
    float h[E], u[E];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if (a.x)
            load_row<R, V>(reinterpret_cast<const R *>(a.x) + at, chunk(c), cols, part(h, c));
        else
#pragma unroll
            for (int e = 0; e < V; ++e) h[c * V + e] = 0.0f;
        if (a.y) load_row<T, V>(reinterpret_cast<const T *>(a.y) + at, chunk(c), cols, part(u, c));
    }
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] *= a.scale;
    if (a.y) {
        float mean, rstd;
        row_stats<NT, E, V>(u, tid, cols, a.post, slots, mean, rstd);
        if (a.stats && tid == 0) {
            a.stats[row] = mean;
            a.stats[(uint64_t)a.rows + row] = rstd;
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float w[V], b[V], g[V];
            if (a.post) load_row<T, V>(a.post_w, chunk(c), cols, w);
            if (a.post == 2) load_row<T, V>(a.post_b, chunk(c), cols, b);
            if (a.gate)
                load_row<T, V>(reinterpret_cast<const T *>(a.gate) + (a.gate_rows > 1 ? at : 0), chunk(c), cols, g);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float v = u[c * V + e];
                if (a.post) v = (v - mean) * rstd * w[e];
                if (a.post == 2) v += b[e];
                if (a.gate) v *= gate_value(a.gate_act, g[e]);
                h[c * V + e] += v;
            }
        }
    } else if (a.stats && tid == 0) {
        a.stats[row] = 0.0f;
        a.stats[(uint64_t)a.rows + row] = 1.0f;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) h[e] = (float)(R)h[e];
    if (a.h)
#pragma unroll
        for (int c = 0; c < C; ++c) store_row<R, V>(reinterpret_cast<R *>(a.h) + at, chunk(c), cols, part(h, c));
    float mean = 0.0f, rstd = 1.0f;
    if (a.n) row_stats<NT, E, V>(h, tid, cols, a.pre, slots + 2 * (NT / 64), mean, rstd);
    if (a.stats && tid == 0) {
        a.stats[2 * (uint64_t)a.rows + row] = mean;
        a.stats[3 * (uint64_t)a.rows + row] = rstd;
    }
    if (!a.n) continue;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        float w[V], b[V], o[V];
        if (a.pre) load_row<T, V>(a.pre_w, chunk(c), cols, w);
        if (a.pre == 2) load_row<T, V>(a.pre_b, chunk(c), cols, b);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            o[e] = h[c * V + e];
            if (a.pre) o[e] = (o[e] - mean) * rstd * w[e];
            if (a.pre == 2) o[e] += b[e];
        }
        store_row<T, V>(reinterpret_cast<T *>(a.n) + at, chunk(c), cols, o);
    }
    }
}

// The backward.  With y^ and h^ the normalised values and <.> the mean over a row:
//   t = dn w_pre,   d = dh + r_h (t - h^ <t h^> - <t>)     (<t> for Layer only)
//   dx = scale d,   du = act(g) d,   dgate = act'(g) d u
//   b = du w_post,  dy = r_y (b - y^ <b y^> - <b>)
// and the column sums of du y^, du, dn h^, dn (and of dgate for one gate row) over the rows.
// A workgroup walks rows blockIdx, blockIdx + grid, ... with its columns' parameters and column
// sums in registers, and writes its sums as one plane of a.work [grid x kPlanes x cols]; the
// next kernel adds the planes.
template <typename T, typename R, int NT, int E>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) unjoin_kernel(UnjoinArgs a) {
    constexpr int V = 16 / sizeof(T), C = E / V;
    constexpr int RPG = NT < 256 ? 256 / NT : 1;
    __shared__ float slots[2][4][NT / 64];
    const uint32_t tid = threadIdx.x % NT, sub = threadIdx.x / NT;
    const uint32_t cols = a.cols;
    const float inv = 1.0f / (float)cols;
    auto chunk = [&](int c) { return ((uint32_t)c * NT + tid) * V; };
    auto part = [&](float (&v)[E], int c) -> float (&)[V] { return *reinterpret_cast<float (*)[V]>(&v[c * V]); };
    float sum[kPlanes][E];
#pragma unroll
    for (int p = 0; p < kPlanes; ++p)
#pragma unroll
        for (int e = 0; e < E; ++e) sum[p][e] = 0.0f;
    uint32_t turn = 0;
    for (uint32_t row = blockIdx.x * RPG + sub; row < a.rows; row += gridDim.x * RPG, turn ^= 1u) {
        const uint64_t at = (uint64_t)row * cols;
        float d[E], hat[E], t[E];
        float s1 = 0.0f, s0 = 0.0f;
        const float h_mean = a.stats[2 * (uint64_t)a.rows + row], h_rstd = a.stats[3 * (uint64_t)a.rows + row];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (a.dh)
                load_row<float, V>(a.dh + at, chunk(c), cols, part(d, c));
            else
#pragma unroll
                for (int e = 0; e < V; ++e) d[c * V + e] = 0.0f;
            if (!a.dn) continue;
            load_row<float, V>(a.dn + at, chunk(c), cols, part(t, c));
            if (!a.pre) continue;
            float w[V];
            load_row<R, V>(reinterpret_cast<const R *>(a.h) + at, chunk(c), cols, part(hat, c));
            load_row<T, V>(a.pre_w, chunk(c), cols, w);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int i = c * V + e;
                hat[i] = (hat[i] - h_mean) * h_rstd;
                sum[2][i] += t[i] * hat[i];
                sum[3][i] += t[i];
                t[i] *= w[e];
                s1 += t[i] * hat[i];
                s0 += t[i];
            }
        }
        if (a.dn) {
            if (a.pre) {
                s1 = row_sum<NT>(s1, slots[turn][0]) * inv;
                s0 = a.pre == 2 ? row_sum<NT>(s0, slots[turn][1]) * inv : 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) d[e] += h_rstd * (t[e] - hat[e] * s1 - s0);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) d[e] += t[e];
            }
        }
        if (a.dx)
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float o[V];
#pragma unroll
                for (int e = 0; e < V; ++e) o[e] = a.scale * d[c * V + e];
                store_row<float, V>(a.dx + at, chunk(c), cols, o);
            }
        if (!a.y) continue;
        // y^ in hat, du in d, then du w_post in t
        const float y_mean = a.stats[row], y_rstd = a.stats[(uint64_t)a.rows + row];
        float t1 = 0.0f, t0 = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float w[V], b[V], g[V], o[V];
            load_row<T, V>(reinterpret_cast<const T *>(a.y) + at, chunk(c), cols, part(hat, c));
            if (a.post) load_row<T, V>(a.post_w, chunk(c), cols, w);
            if (a.post == 2) load_row<T, V>(a.post_b, chunk(c), cols, b);
            if (a.gate)
                load_row<T, V>(reinterpret_cast<const T *>(a.gate) + (a.gate_rows > 1 ? at : 0), chunk(c), cols, g);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int i = c * V + e;
                float u = hat[i];
                if (a.post) {
                    hat[i] = (hat[i] - y_mean) * y_rstd;
                    u = hat[i] * w[e];
                    if (a.post == 2) u += b[e];
                }
                if (a.gate) {
                    const float v = gate_value(a.gate_act, g[e]);
                    o[e] = d[i] * u * gate_slope(a.gate_act, v);
                    sum[4][i] += o[e];
                    d[i] *= v;
                }
                t[i] = d[i];
                if (a.post) {
                    sum[0][i] += d[i] * hat[i];
                    sum[1][i] += d[i];
                    t[i] *= w[e];
                    t1 += t[i] * hat[i];
                    t0 += t[i];
                }
            }
            if (a.gate && a.dgate && a.gate_rows > 1) store_row<float, V>(a.dgate + at, chunk(c), cols, o);
        }
        if (a.post) {
            t1 = row_sum<NT>(t1, slots[turn][2]) * inv;
            t0 = a.post == 2 ? row_sum<NT>(t0, slots[turn][3]) * inv : 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) t[e] = y_rstd * (t[e] - hat[e] * t1 - t0);
        }
        if (a.dy)
#pragma unroll
            for (int c = 0; c < C; ++c) store_row<float, V>(a.dy + at, chunk(c), cols, part(t, c));
    }
    if (!a.work) return;
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
        if (!(a.planes >> p & 1u)) continue;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float *plane = a.work + ((uint64_t)(blockIdx.x * RPG + sub) * kPlanes + p) * cols;
            store_row<float, V>(plane, chunk(c), cols, part(sum[p], c));
        }
    }
}

// Column sums: the planes of a.work added in a fixed order, four slices of planes per column and
// then the slices.  Column sums that the configuration does not have are written as zeros.
__global__ void __launch_bounds__(256) unjoin_sums_kernel(UnjoinArgs a, uint32_t count) {
    __shared__ float part[4][64];
    const uint32_t lane = threadIdx.x & 63u, slice = threadIdx.x >> 6, p = blockIdx.y;
    const uint32_t col = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (col < a.cols && (a.planes >> p & 1u))
        for (uint32_t g = slice; g < count; g += 4) s += a.work[((uint64_t)g * kPlanes + p) * a.cols + col];
    part[slice][lane] = s;
    __syncthreads();
    if (slice || col >= a.cols) return;
    s = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
    if (p < 4) {
        if (a.dparam) a.dparam[(uint64_t)p * a.cols + col] = s;
    } else if (a.gate_sum) {
        a.gate_sum[col] = s;
    }
}

template <typename T, typename R, int NT, int E> hipError_t join_t(const JoinArgs &a, hipStream_t s) {
    constexpr uint32_t rpg = NT < 256 ? 256 / NT : 1;
    const uint32_t groups = (a.rows + rpg - 1) / rpg;
    hipLaunchKernelGGL((join_kernel<T, R, NT, E>), dim3(groups < (1u << 20) ? groups : 1u << 20), dim3(NT < 256 ? 256 : NT), 0, s, a);
    return hipGetLastError();
}

template <typename T, typename R> hipError_t join_c(const JoinArgs &a, hipStream_t s) {
    if (a.cols <= 512) return join_t<T, R, 64, 8>(a, s);
    if (a.cols <= 1024) return join_t<T, R, 64, 16>(a, s);
    if (a.cols <= 2048) return join_t<T, R, 256, 8>(a, s);
    if (a.cols <= 4096) return join_t<T, R, 512, 8>(a, s);
    return join_t<T, R, 1024, 8>(a, s);
}

template <typename T, typename R, int NT, int E> hipError_t unjoin_t(const UnjoinArgs &a, hipStream_t s) {
    constexpr uint32_t rpg = NT < 256 ? 256 / NT : 1;
    const uint32_t planes = residual_planes(a.rows, a.cols);
    hipLaunchKernelGGL((unjoin_kernel<T, R, NT, E>), dim3(planes / rpg), dim3(NT < 256 ? 256 : NT), 0, s, a);
    if (a.work)
        hipLaunchKernelGGL(unjoin_sums_kernel, dim3((a.cols + 63) / 64, kPlanes), dim3(256), 0, s, a, planes);
    return hipGetLastError();
}

template <typename T, typename R> hipError_t unjoin_c(const UnjoinArgs &a, hipStream_t s) {
    if (a.cols <= 512) return unjoin_t<T, R, 64, 8>(a, s);
    if (a.cols <= 2048) return unjoin_t<T, R, 256, 8>(a, s);
    if (a.cols <= 4096) return unjoin_t<T, R, 512, 8>(a, s);
    return unjoin_t<T, R, 512, 16>(a, s);
}

}  // namespace

hipError_t launch_join(const JoinArgs &a, uint32_t dtype, uint32_t stream_dtype, hipStream_t s) {
    if (dtype == 0) return join_c<float, float>(a, s);
    return stream_dtype ? join_c<half_t, half_t>(a, s) : join_c<half_t, float>(a, s);
}

hipError_t launch_unjoin(const UnjoinArgs &a, uint32_t dtype, uint32_t stream_dtype, hipStream_t s) {
    if (dtype == 0) return unjoin_c<float, float>(a, s);
    return stream_dtype ? unjoin_c<half_t, half_t>(a, s) : unjoin_c<half_t, float>(a, s);
}

}  // namespace skl

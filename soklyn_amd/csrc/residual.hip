// residual.hip — the join between two blocks of a residual network, forward and backward:
//
//   u = post(y)                    the norm behind the block (none, RMS, Layer)
//   h = scale x + act(gate) u      the residual stream, rounded to its type
//   n = pre(h)                     the norm before the next block, of h as stored
//
// A row is held in registers from its loads to its stores, so each tensor crosses HBM once, which is
// what bounds both kernels; the norms' sums are two-pass (mean, then squared deviations).
#include <algorithm>

#include "residual.h"
#include "launch.h"
#include "rows.h"

namespace skl {

constexpr float kNormEps = 1e-6f;   // the blocks' own norms add the same

namespace {

__device__ __forceinline__ float gate_value(uint32_t act, float g) {
    if (act == 1) return sigmoid_fast(g);
    if (act == 4) return tanh_fast(g);
    return g;
}
// The gate's slope from its value a.
__device__ __forceinline__ float gate_slope(uint32_t act, float a) {
    if (act == 1) return a * (1.0f - a);
    if (act == 4) return 1.0f - a * a;
    return 1.0f;
}

// Mean and reciprocal deviation of a row's values v (zero past its end).
template <int NT, int E>
__device__ __forceinline__ void row_stats(const float (&v)[E + 1], const RowMap<NT> &map, uint32_t norm, float *slots,
                                          float &mean, float &rstd) {
    mean = 0.0f;
    rstd = 1.0f;
    if (norm == 0) return;
    const float inv = 1.0f / (float)map.cols;
    if (norm == 2) {
        float s[1] = {0.0f};
#pragma unroll
        for (int e = 0; e <= E; ++e) s[0] += v[e];
        row_sums<NT>(s, slots);
        mean = s[0] * inv;
    }
    float q[1] = {0.0f};
#pragma unroll
    for (int e = 0; e <= E; ++e) {
        const float d = (e < E ? map.whole(e / 4) : map.tailed()) ? v[e] - mean : 0.0f;
        q[0] += d * d;
    }
    row_sums<NT>(q, slots + NT / 64);
    rstd = 1.0f / sqrtf(q[0] * inv + kNormEps);
}

// One row per NT threads (several to a workgroup of 256 where a wave, or a quarter, holds one).
// 8192 x 4096, fp16 with an fp32 stream, a gate for each row, RMS on both sides: 470 MB in 94.8 us,
// 4.96 TB/s, of 5.1 for a large copy; one row of it 4.6 us, loads and two sums one behind the other.
// Wider rows, one on each workgroup of 512, are further from it (RMS, one gate): 4096 x 8192 fp16
// 83 us, 3.2 TB/s, fp32 126, 4.3 TB/s; 8192 x 5120, where three eighths of the threads' vectors are empty,
// 168 and 169 us, 2.0 and 4.0 TB/s.
template <typename T, typename R, int NT, int E>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) join_kernel(JoinArgs a) {
    constexpr int RPG = NT < 256 ? 256 / NT : 1;
    constexpr int S = NT < 64 ? 1 : NT / 64;
    __shared__ float both[2][4 * S];   // in turns: a row may have one sum, and so one barrier
    const RowMap<NT> map{threadIdx.x % NT, a.cols};
    uint32_t turn = 0;
    const uint32_t step = gridDim.x * RPG;
    for (uint32_t row = blockIdx.x * RPG + sub_row<NT>(); row < a.rows; row = next_row(row, step, a.rows), turn ^= 1u) {
        float *slots = both[turn];
        const uint64_t at = (uint64_t)row * a.cols;
        float mean = 0.0f, rstd = 1.0f;
        RowPart<R, E> x;
        RowPart<T, E> y, g;
        if (a.x) map.template read<R, E>(reinterpret_cast<const R *>(a.x) + at, x);
        if (a.y) map.template read<T, E>(reinterpret_cast<const T *>(a.y) + at, y);
        if (a.gate) map.template read<T, E>(reinterpret_cast<const T *>(a.gate) + (a.gate_rows > 1 ? at : 0), g);
        float h[E + 1];
        if (a.x) {
            map.template floats<R, E>(x, h);
#pragma unroll
            for (int e = 0; e <= E; ++e) h[e] *= a.scale;
        } else {
#pragma unroll
            for (int e = 0; e <= E; ++e) h[e] = 0.0f;
        }
        if (a.y) {
            float u[E + 1];
            map.template floats<T, E>(y, u);
            row_stats<NT, E>(u, map, a.post, slots, mean, rstd);
            if (a.post) {
                float w[E + 1];
                map.template read<T, E>(a.post_w, w);
#pragma unroll
                for (int e = 0; e <= E; ++e) u[e] = (u[e] - mean) * rstd * w[e];
                if (a.post == 2) {
                    map.template read<T, E>(a.post_b, w);
#pragma unroll
                    for (int e = 0; e <= E; ++e) u[e] += w[e];
                }
            }
            if (a.gate) {
                float v[E + 1];
                map.template floats<T, E>(g, v);
#pragma unroll
                for (int e = 0; e <= E; ++e) u[e] *= gate_value(a.gate_act, v[e]);
            }
#pragma unroll
            for (int e = 0; e <= E; ++e) h[e] += u[e];
        }
        if (a.stats && map.tid == 0) {
            a.stats[row] = mean;
            a.stats[(uint64_t)a.rows + row] = rstd;
        }
#pragma unroll
        for (int e = 0; e <= E; ++e) h[e] = (float)(R)h[e];
        if (a.h) map.template write<R, E>(reinterpret_cast<R *>(a.h) + at, h);
        mean = 0.0f;
        rstd = 1.0f;
        if (a.n) row_stats<NT, E>(h, map, a.pre, slots + 2 * S, mean, rstd);
        if (a.stats && map.tid == 0) {
            a.stats[2 * (uint64_t)a.rows + row] = mean;
            a.stats[3 * (uint64_t)a.rows + row] = rstd;
        }
        if (!a.n) continue;
        if (a.pre) {
            // past the row's end w is 0, and what is there is not written
            float w[E + 1];
            map.template read<T, E>(a.pre_w, w);
#pragma unroll
            for (int e = 0; e <= E; ++e) h[e] = (h[e] - mean) * rstd * w[e];
            if (a.pre == 2) {
                map.template read<T, E>(a.pre_b, w);
#pragma unroll
                for (int e = 0; e <= E; ++e) h[e] += w[e];
            }
        }
        map.template write<T, E>(reinterpret_cast<T *>(a.n) + at, h);
    }
}

// The backward.  With y^ and h^ the normalised values and <.> the mean over a row:
//   t = dn w_pre,   d = dh + r_h (t - h^ <t h^> - <t>)     (<t> for Layer only)
//   dx = scale d,   du = act(g) d,   dgate = act'(g) d u
//   b = du w_post,  dy = r_y (b - y^ <b y^> - <b>)
// and the column sums of du y^, du, dn h^, dn (and of dgate for one gate row) over the rows.
// A workgroup walks rows blockIdx, blockIdx + grid, ... with its column sums in registers and the
// next row's tensors on their way, and writes its sums as one plane of a.work [grid x kPlanes x
// cols]; the next kernel adds the planes: 16384 x 2048 fp16, 671 MB in 137 + 6 us, 4.7 TB/s.  BIAS: a Layer norm is there, so that du and dn are summed.
// Rows of more than 4096 columns: the sums but dn's, which do not fit the registers, are in LDS, each
// thread its own, and a row's tensors are loaded where they are used, not a row ahead (of 256 registers BIAS
// takes 236 to 244, the other form 192 to 200).  One workgroup to a CU then waits for dn and h, for dh
// and for y: 4096 x 8192 fp16 with RMS on both sides 177 us, with Layer 191 (floor 131 at 5.12 TB/s),
// fp32 193 and 207 (157); 8192 x 5120 fp16 245 and 264 (164), fp32 258 and 279 (197).
template <typename T, typename R, int NT, int E, bool BIAS>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) unjoin_kernel(UnjoinArgs a) {
    constexpr int RPG = NT < 256 ? 256 / NT : 1, S = NT < 64 ? 1 : NT / 64;
    __shared__ float slots[2][4 * S];
    __shared__ float join[RPG > 1 ? RPG : 1][RPG > 1 ? NT * E + 4 : 1];
    const uint32_t sub = sub_row<NT>();
    const RowMap<NT> map{threadIdx.x % NT, a.cols};
    const float inv = 1.0f / (float)a.cols;
    constexpr bool kWide = E * NT > 4096;
    constexpr int kKept = BIAS ? 4 : 3;   // 32 KB each
    __shared__ f32x4 kept[kWide ? kKept : 1][kWide ? E / 4 : 1][kWide ? NT : 1];
    float sum[kPlanes][E + 1];
#pragma unroll
    for (int p = 0; p < kPlanes; ++p)
#pragma unroll
        for (int e = 0; e <= E; ++e) sum[p][e] = 0.0f;
    if constexpr (kWide)
#pragma unroll
        for (int i = 0; i < kKept * (E / 4); ++i) kept[i / (E / 4)][i % (E / 4)][threadIdx.x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // adds v to column sum p
    auto add = [&](int p, const float (&v)[E + 1]) {
        if (kWide && p != 3) {
#pragma unroll
            for (int c = 0; c < E / 4; ++c) {
                f32x4 &k = kept[p == 1 ? 3 : p / 2][c][threadIdx.x];
                k += f32x4{v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]};
            }
            sum[p][E] += v[E];
        } else {
#pragma unroll
            for (int e = 0; e <= E; ++e) sum[p][e] += v[e];
        }
    };
    struct Parts {
        RowPart<float, E> dn, dh;
        RowPart<R, E> h;
        RowPart<T, E> y;
    } in;
    auto read = [&](uint32_t row) {
        const uint64_t at = (uint64_t)row * a.cols;
        if (a.dn) map.template read<float, E>(a.dn + at, in.dn);
        if (!kWide && a.dh) map.template read<float, E>(a.dh + at, in.dh);
        if (a.pre) map.template read<R, E>(reinterpret_cast<const R *>(a.h) + at, in.h);
        if (!kWide && a.y) map.template read<T, E>(reinterpret_cast<const T *>(a.y) + at, in.y);
    };
    uint32_t turn = 0, row = blockIdx.x * RPG + sub;
    const uint32_t step = gridDim.x * RPG;
    if (!kWide && row < a.rows) read(row);
    for (; row < a.rows; row = next_row(row, step, a.rows), turn ^= 1u) {
        const uint64_t at = (uint64_t)row * a.cols;
        float d[E + 1], t[E + 1], hat[E + 1], y[E + 1];
        if constexpr (kWide) read(row);
        // from behind the join, once the sums of what comes from the next block are taken
        auto behind = [&] {
            if (kWide && a.dh)
                map.template read<float, E>(a.dh + at, d);
            else if (a.dh)
                map.template floats<float, E>(in.dh, d);
            else
#pragma unroll
                for (int e = 0; e <= E; ++e) d[e] = 0.0f;
        };
        if constexpr (!kWide) behind();
        if (a.dn) map.template floats<float, E>(in.dn, t);
        if (a.pre) map.template floats<R, E>(in.h, hat);
        if (!kWide && a.y) map.template floats<T, E>(in.y, y);
        if (!kWide && step < a.rows - row) read(row + step);
        if (a.dn && a.pre) {
            const float mean = a.stats[2 * (uint64_t)a.rows + row], rstd = a.stats[3 * (uint64_t)a.rows + row];
            float w[E + 1], s[2] = {0.0f, 0.0f};
            map.template read<T, E>(a.pre_w, w);
            float product[E + 1];
#pragma unroll
            for (int e = 0; e <= E; ++e) {
                hat[e] = (hat[e] - mean) * rstd;
                product[e] = t[e] * hat[e];
            }
            add(2, product);
            if constexpr (BIAS) add(3, t);
#pragma unroll
            for (int e = 0; e <= E; ++e) {
                t[e] *= w[e];   // 0 past the row's end
                s[0] += t[e] * hat[e];
                s[1] += t[e];
            }
            row_sums<NT>(s, slots[turn]);
            s[0] *= inv;
            s[1] = a.pre == 2 ? s[1] * inv : 0.0f;
            if constexpr (kWide) behind();
#pragma unroll
            for (int e = 0; e <= E; ++e) d[e] += rstd * (t[e] - hat[e] * s[0] - s[1]);
        } else {
            if constexpr (kWide) behind();
            if (a.dn)
#pragma unroll
                for (int e = 0; e <= E; ++e) d[e] += t[e];
        }
        if (a.dx) {
#pragma unroll
            for (int e = 0; e <= E; ++e) t[e] = a.scale * d[e];
            map.template write<float, E>(a.dx + at, t);
        }
        if (!a.y) continue;
        const float mean = a.stats[row], rstd = a.stats[(uint64_t)a.rows + row];
        if constexpr (kWide) map.template read<T, E>(reinterpret_cast<const T *>(a.y) + at, y);
        float w[E + 1];
        if (a.post) {
            map.template read<T, E>(a.post_w, w);
#pragma unroll
            for (int e = 0; e <= E; ++e) y[e] = (y[e] - mean) * rstd;
        }
        if (a.gate) {
            float u[E + 1];
#pragma unroll
            for (int e = 0; e <= E; ++e) u[e] = a.post ? y[e] * w[e] : y[e];
            if (BIAS && a.post == 2) {
                map.template read<T, E>(a.post_b, t);
#pragma unroll
                for (int e = 0; e <= E; ++e) u[e] += t[e];
            }
            map.template read<T, E>(reinterpret_cast<const T *>(a.gate) + (a.gate_rows > 1 ? at : 0), t);
#pragma unroll
            for (int e = 0; e <= E; ++e) {
                const float v = gate_value(a.gate_act, t[e]);
                u[e] = d[e] * u[e] * gate_slope(a.gate_act, v);
                d[e] *= v;
            }
            if (a.gate_sum) add(4, u);
            if (a.dgate) map.template write<float, E>(a.dgate + at, u);
        }
        if (a.post) {
            float s[2] = {0.0f, 0.0f}, product[E + 1];
#pragma unroll
            for (int e = 0; e <= E; ++e) product[e] = d[e] * y[e];
            add(0, product);
            if constexpr (BIAS) add(1, d);
#pragma unroll
            for (int e = 0; e <= E; ++e) {
                d[e] *= w[e];
                s[0] += d[e] * y[e];
                s[1] += d[e];
            }
            row_sums<NT>(s, slots[turn] + 2 * S);
            s[0] *= inv;
            s[1] = a.post == 2 ? s[1] * inv : 0.0f;
#pragma unroll
            for (int e = 0; e <= E; ++e) d[e] = rstd * (d[e] - y[e] * s[0] - s[1]);
        }
        if (a.dy) map.template write<float, E>(a.dy + at, d);
    }
    if (!a.work) return;
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
        if (!(a.planes >> p & 1u)) continue;
        if (kWide && p != 3 && (BIAS || p != 1))
#pragma unroll
            for (int e = 0; e < E; ++e) sum[p][e] = kept[p == 1 ? 3 : p / 2][e / 4][threadIdx.x][e % 4];
        float *plane = a.work + ((uint64_t)blockIdx.x * kPlanes + p) * a.cols;
        if constexpr (RPG == 1) {
            map.template write<float, E>(plane, sum[p]);
        } else {
            __syncthreads();
            map.template write<float, E>(join[sub], sum[p]);
            __syncthreads();
            for (uint32_t col = threadIdx.x; col < a.cols; col += 256) {
                float s = 0.0f;
#pragma unroll
                for (int i = 0; i < RPG; ++i) s += join[i][col];
                plane[col] = s;
            }
        }
    }
}

// Column sums: the planes of a.work added in a fixed order, 32 slices of them per column and then
// the slices.  Column sums that the configuration does not have are written as zeros.
__global__ void __launch_bounds__(1024) unjoin_sums_kernel(UnjoinArgs a, uint32_t count) {
    __shared__ float part[32][33];
    const uint32_t lane = threadIdx.x & 31u, slice = threadIdx.x >> 5, p = blockIdx.y;
    const uint32_t col = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (col < a.cols && (a.planes >> p & 1u))
#pragma unroll 8
        for (uint32_t g = slice; g < count; g += 32) s += a.work[((uint64_t)g * kPlanes + p) * a.cols + col];
    part[slice][lane] = s;
    __syncthreads();
    if (slice || col >= a.cols) return;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += part[i][lane];
    if (p < 4) {
        if (a.dparam) a.dparam[(uint64_t)p * a.cols + col] = s;
    } else if (a.gate_sum) {
        a.gate_sum[col] = s;
    }
}

template <typename T, typename R, int NT, int E> hipError_t join_t(const JoinArgs &a, hipStream_t s) {
    constexpr uint32_t rpg = NT < 256 ? 256 / NT : 1;
    const uint32_t groups = (a.rows - 1) / rpg + 1;
    hipLaunchKernelGGL((join_kernel<T, R, NT, E>), dim3(groups < (1u << 20) ? groups : 1u << 20),
                       dim3(NT < 256 ? 256 : NT), 0, s, a);
    return hipGetLastError();
}

template <typename T, typename R> hipError_t join_c(const JoinArgs &a, hipStream_t s) {
    if (a.cols <= 64) return join_t<T, R, 16, 4>(a, s);
    if (a.cols <= 256) return join_t<T, R, 64, 4>(a, s);
    if (a.cols <= 1024) return join_t<T, R, 64, 16>(a, s);
    if (a.cols <= 2048) return join_t<T, R, 256, 8>(a, s);
    if (a.cols <= 4096) return join_t<T, R, 256, 16>(a, s);
    return join_t<T, R, 512, 16>(a, s);
}

// Workgroups of `kernel` that the current GPU holds at once.
template <class K> uint32_t resident(K kernel, int threads) {
    int dev = 0, cus = 0, per_cu = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kernel, threads, 0) != hipSuccess || cus * per_cu <= 0)
        return 256;
    return (uint32_t)(cus * per_cu);
}

// As many workgroups as the GPU holds at once, each with as many rows as the next (16384 x 2048
// fp16: 150 us on 768 workgroups, three to a CU; 175 on 512, 183 on 1024); two rows at least once
// there is one for every CU, which halves the planes (500 x 777 fp32: 14.4 and 15.6 us).
template <typename T, typename R, int NT, int E, bool BIAS> hipError_t unjoin_t(const UnjoinArgs &a, hipStream_t s) {
    constexpr uint32_t rpg = NT < 256 ? 256 / NT : 1, threads = NT < 256 ? 256 : NT;
    static const uint32_t held = resident(unjoin_kernel<T, R, NT, E, BIAS>, threads);
    const uint32_t groups = (a.rows - 1) / rpg + 1, most = std::min(held, residual_planes(a.rows, a.cols));
    const uint32_t each = std::max((groups - 1) / most + 1, groups > 256 ? 2u : 1u);
    const uint32_t grid = (groups - 1) / each + 1;
    hipLaunchKernelGGL((unjoin_kernel<T, R, NT, E, BIAS>), dim3(grid), dim3(threads), 0, s, a);
    if (a.work)
        hipLaunchKernelGGL(unjoin_sums_kernel, dim3((a.cols + 31) / 32, kPlanes), dim3(1024), 0, s, a, grid);
    return hipGetLastError();
}

template <typename T, typename R, int NT, int E> hipError_t unjoin_n(const UnjoinArgs &a, hipStream_t s) {
    return a.pre == 2 || a.post == 2 ? unjoin_t<T, R, NT, E, true>(a, s) : unjoin_t<T, R, NT, E, false>(a, s);
}

template <typename T, typename R> hipError_t unjoin_c(const UnjoinArgs &a, hipStream_t s) {
    if (a.cols <= 64) return unjoin_n<T, R, 16, 4>(a, s);
    if (a.cols <= 256) return unjoin_n<T, R, 64, 4>(a, s);
    if (a.cols <= 512) return unjoin_n<T, R, 64, 8>(a, s);
    if (a.cols <= 1024) return unjoin_n<T, R, 256, 4>(a, s);
    if (a.cols <= 2048) return unjoin_n<T, R, 256, 8>(a, s);
    if (a.cols <= 4096) return unjoin_n<T, R, 512, 8>(a, s);
    return unjoin_n<T, R, 512, 16>(a, s);
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

// distill.hip — the error of an output layer that learns from a teacher's top logits.  Per row,
// with z the layer's logits, v_j at class i_j the teacher's (j over the row's held slots), t the
// temperature and y the label:
//
//   q = softmax_j(v / t), added up over the slots of each class,  p = softmax(z / t),  p1 = softmax(z)
//   loss = alpha t^2 sum_c q_c (log q_c - log p_c) - (1 - alpha) log p1[y]
//   d loss / d z = alpha t (p - q) + (1 - alpha) (p1 - [y])
//
// the gradient times the loss scale into grad and d_prenorm (and its fp16 copy).  A row without
// held slots has no first term, one without a label no second, and one whose logits are all -inf
// neither; NaN and +inf logits make their row NaN, as in a softmax.
#include <type_traits>

#include "distill.h"
#include "launch.h"
#include "rows.h"

namespace skl {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int V = 4;   // columns of a vector

// Orders a row's LDS accesses among its NT threads; a wave's own are executed in order.
template <int NT> __device__ __forceinline__ void row_sync() {
    if constexpr (NT > 64) {
        __syncthreads();
    } else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

__device__ __forceinline__ uint32_t opaque(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}

// LDS words of one row: the columns' shares where they have a table, marks, four words per slot, and without
// a table the slots that found their mark made, and their classes.
__host__ __device__ constexpr uint32_t distill_marks(int NT, bool table) {
    return NT == 16 ? 8 : NT == 64 ? 64 : table ? 128 : 256;
}
__host__ __device__ constexpr uint32_t distill_words(int NT, int E, bool table, uint32_t top) {
    return distill_marks(NT, table) + (table ? NT * E + 4 * top : 6 * top + 1);
}

// NT threads to a row (16 or 64: several rows to a workgroup of 256).  They hold it in registers, E
// elements each, from one read; MORE: what is longer than that is read for the maximum, for each of the two
// sums that the row needs, and for the gradient: up to four times.
//
// What the teacher takes off a column.  TABLE: a table of the columns in LDS, filled by the slots (a
// class that two of them name is seen when the second sets its bit in marks; then each slot looks
// through all of them and adds up those of its class, in their order).  Otherwise marks has
// a bit for each 2^group columns that says whether a slot may be among them; the slots of a marked
// vector are found by its whole wave, a slot to a lane.  2048 rows of 50257 classes with 64 slots:
// 588 us when each lane looked through the slots by itself, 286 us so.  There only the loss asks
// whether a class repeats: slots that found their group marked go on a list, and each slot looks
// through that (512 rows of 50257 fp16 with 1000 slots, no two alike: 696 us, 694 without the question
// and 1002 when each of those looked through all slots; with two alike in half of the rows 790).
//
// HBM bounds long rows (fp16: 2 bytes of a logit read, 10 written): 8192 rows of 8000 take 150 us,
// 5.2 TB/s, 4096 of 30000 308 us, 4.8 TB/s, 2048 of 50257 274 us, 4.5 TB/s (there two workgroups to a
// CU instead of one, with 64 registers a thread, are not ahead: 294 us against 288 in one run).  MORE,
// with 64 slots, teacher alone and with labels: 1024 rows of 128256 fp16 380 and 410 us (floor 308 at a
// large copy's 5.12 TB/s), 512 of 256000 520 and 585 (307), fp32 485 and 512, 561 and 630: the reads past
// the first.  Few short rows are launch and latency: 1024 rows of 1000 8.2 us.
//
// A softmax's exponent is (z - max) k and not fma(z, k, -max k): the rounding of max k is the same in
// every term, but past 2^31 (large logits, a small temperature) takes the largest term itself out of
// range.
template <typename T, int NT, int E, bool TABLE, bool MORE>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) distill_kernel(DistillArgs a) {
    constexpr int W = NT / 64, C = E / V, RPG = NT < 256 ? 256 / NT : 1, LANES = NT < 64 ? NT : 64;
    constexpr uint32_t kMarks = distill_marks(NT, TABLE);
    typedef typename Unaligned<T, V>::type Vec;
    extern __shared__ f32x4 lds[];
    __shared__ float red[3][W > 0 ? W : 1];
    const uint32_t tid = threadIdx.x % NT, lane = threadIdx.x % LANES, n = a.n, top = a.top;
    float *table = reinterpret_cast<float *>(lds) + sub_row<NT>() * distill_words(NT, E, TABLE, top);
    uint32_t *marks = reinterpret_cast<uint32_t *>(table + (TABLE ? NT * E : 0));
    int32_t *at = reinterpret_cast<int32_t *>(marks + kMarks);
    float *value = reinterpret_cast<float *>(at + top), *q = value + top, *z_at = q + top;
    uint32_t *late = reinterpret_cast<uint32_t *>(z_at + top);   // without a table: their number, slots and classes
    const float k_soft = kLog2e / a.tau;
    uint32_t group = TABLE ? 0 : 2;   // without a table a vector lies in one group
    if constexpr (!TABLE)
        while ((n + V - 1) >> group >= kMarks * 32u) ++group;

    for (uint32_t row = blockIdx.x * RPG + sub_row<NT>(); row < a.rows; row = next_row(row, gridDim.x * RPG, a.rows)) {
        const uint64_t row_at = (uint64_t)row * n;
        // A row of an odd width starts anywhere.  Its threads take its vectors from the last of the
        // matrix's own vectors that begins at or before it, so that every whole one is aligned if
        // the matrix is: the row's elements are at positions [lo, hi) of what begins lo before it.
        const uint32_t lo = (uint32_t)(row_at % V), hi = lo + n;
        const T *z = reinterpret_cast<const T *>(a.logits) + (row_at - lo);
        // whole vectors [v0, v1); what is cut off the first and last of the row goes to threads 0 and 1
        const uint32_t v0 = lo ? 1 : 0, v1 = hi / V;
        const bool edged = tid == 0 ? lo != 0 : tid == 1 && v1 >= v0 && hi % V;
        const uint32_t edge_p = tid == 0 ? 0 : v1 * V;
        float edge[V];
#pragma unroll
        for (int e = 0; e < V; ++e) edge[e] = edged && edge_p + e >= lo && edge_p + e < hi ? to_f32(z[edge_p + e]) : -INFINITY;
        Vec held[C];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const uint32_t i = opaque(c * NT + tid);
#pragma unroll
            for (int e = 0; e < V; ++e) held[c][e] = (T)-INFINITY;
            if (i >= v0 && i < v1) held[c] = *reinterpret_cast<const Vec *>(z + i * V);
        }
        // f(position, values, whole) over the row, -inf where there is nothing, by whole waves.  The
        // registers are opaque to each pass, or the compiler would keep one pass's exponentials and
        // positions for the next and spill.
        auto each = [&](auto f) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                asm volatile("" : "+v"(held[c]));
                if ((uint32_t)c * NT >= v1) break;
                float v[V];
#pragma unroll
                for (int e = 0; e < V; ++e) v[e] = (float)held[c][e];
                f(opaque(c * NT + tid) * V, v, std::true_type());
                if constexpr (C > 4) __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (MORE)
                for (uint32_t i0 = C * NT; i0 < v1; i0 += NT) {
                    const uint32_t i = i0 + tid;
                    float v[V];
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] = -INFINITY;
                    if (i >= v0 && i < v1) {
                        const Vec w = *reinterpret_cast<const Vec *>(z + i * V);
#pragma unroll
                        for (int e = 0; e < V; ++e) v[e] = (float)w[e];
                    }
                    f(i * V, v, std::true_type());
                }
            f(edge_p, edge, std::false_type());
        };

        // the teacher's slots and the label
        for (uint32_t j = tid; j < kMarks; j += NT) marks[j] = 0;
        if (!TABLE && tid == 0) late[0] = 0;
        if constexpr (TABLE)
#pragma unroll
            for (int c = 0; c < C; ++c) reinterpret_cast<f32x4 *>(table)[c * NT + tid] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
        for (uint32_t j = tid; j < top; j += NT) {
            const int32_t i = a.index[(uint64_t)row * top + j];
            const float v = a.value[(uint64_t)row * top + j];
            const bool in = (uint32_t)i < n;
            at[j] = in ? i : -1;
            value[j] = in ? v : -INFINITY;
            z_at[j] = in ? to_f32(z[lo + i]) : 0.0f;
        }
        const int32_t y = a.label ? a.label[row] : -1;
        const bool labelled = (uint32_t)y < n;
        const float z_y = labelled ? to_f32(z[lo + y]) : 0.0f;
        row_sync<NT>();
        // each group of lanes for itself, in one order: the largest logit, then the sum
        float t_max = -INFINITY, t_sum = 0.0f;
#pragma unroll 1
        for (uint32_t j = lane; j < top; j += LANES) t_max = fmaxf(t_max, value[j]);
        t_max = lanes_max<LANES>(t_max);
        t_max = t_max == -INFINITY ? 0.0f : t_max;
#pragma unroll 1
        for (uint32_t j = lane; j < top; j += LANES)
            t_sum += at[j] >= 0 ? __builtin_amdgcn_exp2f((value[j] - t_max) * k_soft) : 0.0f;
        t_sum = lanes_sum<LANES>(t_sum);
        const bool taught = a.alpha > 0.0f && t_sum != 0.0f;   // NaN: taught, and NaN
        bool twice = false;
#pragma unroll 1
        for (uint32_t j = tid; j < top; j += NT) {
            const uint32_t b = ((uint32_t)at[j] + (TABLE ? 0 : lo)) >> group, bit = 1u << (b & 31u);
            q[j] = taught && at[j] >= 0 ? __builtin_amdgcn_exp2f((value[j] - t_max) * k_soft) / t_sum : 0.0f;
            if (at[j] >= 0 && (atomicOr(&marks[b >> 5], bit) & bit)) {
                twice = TABLE || a.loss;
                if (!TABLE && a.loss) {
                    uint32_t *entry = late + 1 + 2 * atomicAdd(&late[0], 1u);
                    entry[0] = j;
                    entry[1] = (uint32_t)at[j];
                }
            }
        }
        if constexpr (!TABLE) {
            const uint32_t b = ((uint32_t)y + lo) >> group;
            if (tid == 0 && labelled) atomicOr(&marks[b >> 5], 1u << (b & 31u));
        }

        // the layer's maximum and sums
        float m = -INFINITY;
        each([&](uint32_t, const float (&v)[V], auto) { m = fmaxf(fmaxf(m, fmaxf(v[0], v[1])), fmaxf(v[2], v[3])); });
        m = lanes_max<LANES>(m);
        if constexpr (NT > 64) {
            if (lane == 0) red[0][tid >> 6] = m;
            twice = __syncthreads_or(twice);   // q and marks too
#pragma unroll
            for (int w = 0; w < W; ++w) m = fmaxf(m, red[0][w]);
        } else {
            twice = __any(twice);
            row_sync<NT>();
        }
        // Without a table, where only the loss asks, a slot's group may have been marked by a neighbour: is
        // there another slot of its class?
        if (!TABLE && twice) {
            uint32_t apart = 1;   // 0: no
            const uint32_t found = late[0];
#pragma unroll 1
            for (uint32_t j = tid; j < top; j += NT) {
                const uint32_t of = (uint32_t)at[j];
#pragma unroll 4
                for (uint32_t i = 0; i < found; ++i)
                    apart = min(apart, late[1 + 2 * i] == j ? 1u : late[2 + 2 * i] ^ of);
            }
            twice = __syncthreads_or(apart == 0);
        }
        const float base = m == -INFINITY ? 0.0f : m;
        if (!twice) {
#pragma unroll 1
            for (uint32_t j = tid; j < top; j += NT) {
                if (TABLE && at[j] >= 0) table[lo + at[j]] = q[j];
                z_at[j] -= base;
            }
        }
        // A class that several slots name has the sum of their shares.  The loss counts each slot with its own
        // share and the logarithm of its class's: by how much that is above its own goes off the class's z.
        // (Below 2^-126, where logarithms end, a share has no part in the loss.)
        if (twice) {
#pragma unroll 1
            for (uint32_t j = tid; j < top; j += NT) {
                const int32_t of = at[j];
                float sum = 0.0f;   // the same, to the bit, for every slot of the class
#pragma unroll 4
                for (uint32_t i = 0; i < top; ++i) sum += at[i] == of ? q[i] : 0.0f;
                if (TABLE && of >= 0) table[lo + of] = sum;
                const float more = __builtin_amdgcn_logf(sum) - __builtin_amdgcn_logf(q[j]);
                z_at[j] = (z_at[j] - base) - (q[j] >= 0x1p-126f ? a.tau * kLn2 * more : 0.0f);
            }
        }
        float s_soft = 0.0f, s_hard = 0.0f;
        if (taught)
            each([&](uint32_t, const float (&v)[V], auto) {
#pragma unroll
                for (int e = 0; e < V; ++e) s_soft += __builtin_amdgcn_exp2f((v[e] - base) * k_soft);
            });
        if (labelled)
            each([&](uint32_t, const float (&v)[V], auto) {
#pragma unroll
                for (int e = 0; e < V; ++e) s_hard += __builtin_amdgcn_exp2f((v[e] - base) * kLog2e);
            });
        s_soft = lanes_sum<LANES>(s_soft);
        s_hard = lanes_sum<LANES>(s_hard);
        if constexpr (NT > 64) {
            if (lane == 0) {
                red[1][tid >> 6] = s_soft;
                red[2][tid >> 6] = s_hard;
            }
            __syncthreads();   // the table too
            s_soft = s_hard = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                s_soft += red[1][w];
                s_hard += red[2][w];
            }
        } else {
            row_sync<NT>();
        }
        // a sum of 0: all logits -inf
        const bool soft = taught && s_soft != 0.0f, hard = labelled && s_hard != 0.0f;
        const float g_soft = soft ? kLossScale * a.alpha * a.tau : 0.0f;
        const float g_hard = hard ? kLossScale * (1.0f - a.alpha) : 0.0f;
        const float w_soft = soft ? g_soft / s_soft : 0.0f, w_hard = hard ? g_hard / s_hard : 0.0f;

        constexpr bool kLane = !TABLE && E < 128;   // two registers that the others do not have
        const int32_t at_lane = kLane && lane < top ? at[lane] : -1;
        const float q_lane = kLane && lane < top ? q[lane] : 0.0f;
        each([&](uint32_t p, const float (&v)[V], auto whole) {
            const bool mine = decltype(whole)::value ? p >= v0 * V && p < v1 * V : edged;
            float g[V];
#pragma unroll
            for (int e = 0; e < V; ++e) g[e] = soft ? w_soft * __builtin_amdgcn_exp2f((v[e] - base) * k_soft) : 0.0f;
            if (hard)
#pragma unroll
                for (int e = 0; e < V; ++e) g[e] += w_hard * __builtin_amdgcn_exp2f((v[e] - base) * kLog2e);
            if constexpr (TABLE) {
                if (!mine) return;
                const f32x4 share = *reinterpret_cast<const f32x4 *>(table + p);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    if (soft) g[e] -= g_soft * share[e];
                    g[e] -= hard && (uint32_t)y + lo == p + e ? g_hard : 0.0f;
                }
            } else {
                const uint32_t b = p >> group;
                uint64_t marked = __ballot(mine && (marks[b >> 5] >> (b & 31u) & 1u));
                while (marked) {
                    const int of = __builtin_ctzll(marked);
                    marked &= marked - 1;
                    const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)p, of);
                    for (uint32_t j = 0; soft && j < top; j += 64) {
                        const int32_t i = kLane && j == 0 ? at_lane : j + lane < top ? at[j + lane] : -1;
                        const float share = g_soft * (kLane && j == 0 ? q_lane : j + lane < top ? q[j + lane] : 0.0f);
                        const uint32_t off = i < 0 ? V : (uint32_t)i + lo - first;
                        uint64_t hits = __ballot(off < V);
                        while (hits) {
                            const int hit = __builtin_ctzll(hits);
                            hits &= hits - 1;
                            const int e_hit = __builtin_amdgcn_readlane((int)off, hit);
                            const float s_hit = lane_of(share, hit);
#pragma unroll
                            for (int e = 0; e < V; ++e) g[e] -= (int)lane == of && e == e_hit ? s_hit : 0.0f;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < V; ++e) g[e] -= (int)lane == of && hard && (uint32_t)y + lo == p + e ? g_hard : 0.0f;
                }
                if (!mine) return;
            }
            auto store = [&](auto *to) {
                typedef std::remove_reference_t<decltype(*to)> S;
                to += row_at - lo;
                if constexpr (decltype(whole)::value) {
                    typename Unaligned<S, V>::type w;
#pragma unroll
                    for (int e = 0; e < V; ++e) w[e] = (S)g[e];
                    *reinterpret_cast<typename Unaligned<S, V>::type *>(to + p) = w;
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (p + e >= lo && p + e < hi) to[p + e] = (S)g[e];
                }
            };
            store(a.grad);
            store(a.d_prenorm);
            if constexpr (sizeof(T) == 2) store(a.d_prenorm_h);
        });

        if (a.loss && tid < 64) {
            // in units of the logits, not of the exponents: these may pass fp32 where the loss does not
            float l = 0.0f;
            const float logs = a.tau * kLn2 * (__builtin_amdgcn_logf(s_soft) - __builtin_amdgcn_logf(t_sum));
            if (soft)   // (opaque: addresses that are kept from the other loops take registers)
#pragma unroll 1
                for (uint32_t j = opaque(lane); j < top; j += LANES)
                    if (q[j] != 0.0f) l += q[j] * (((value[j] - t_max) - z_at[j]) + logs);
            l = lanes_sum<LANES>(l) * (a.alpha * a.tau);
            if (hard) l -= (1.0f - a.alpha) * ((z_y - base) - kLn2 * __builtin_amdgcn_logf(s_hard));
            if (lane == 0) a.loss[row] = l;
        }
        row_sync<NT>();   // the next row's slots
    }
}

template <typename T, int NT, int E, bool TABLE, bool MORE = false> hipError_t distill_t(const DistillArgs &a, hipStream_t s) {
    constexpr uint32_t rpg = NT < 256 ? 256 / NT : 1;
    const uint32_t groups = (a.rows - 1) / rpg + 1;
    hipLaunchKernelGGL((distill_kernel<T, NT, E, TABLE, MORE>), dim3(groups < (1u << 20) ? groups : 1u << 20),
                       dim3(NT < 256 ? 256 : NT), rpg * distill_words(NT, E, TABLE, a.top) * 4, s, a);
    return hipGetLastError();
}

// The row and up to three columns before it have to fit.  Few threads with many elements each are
// ahead, as long as the rows fill the GPU: 16384 rows of 1000 fp16 classes take 50 us a wave to a
// row, 83 us a workgroup to a row; 1024 rows of them 11.6 and 9.9 us.  8192 rows of 8000: 165 us on
// 256 threads, 211 on 512, 283 on 1024.  Past 32768 columns the registers of two workgroups of 512
// no longer fit a CU: 2048 rows of 50257, 287 us on 1024 threads, 310 on 512.
template <typename T> hipError_t distill_n(const DistillArgs &a, hipStream_t s) {
    const uint32_t n = a.n + 3;
    const bool few = a.rows < 4096 || a.top > 64;   // the slots of several rows would crowd the LDS
    if (n <= 64 && a.top <= 64) return distill_t<T, 16, 4, true>(a, s);
    if (n <= 256 && a.top <= 64) return distill_t<T, 16, 16, true>(a, s);
    if (n <= 1024 && few) return distill_t<T, 256, 4, true>(a, s);
    if (n <= 512) return distill_t<T, 64, 8, true>(a, s);
    if (n <= 1024) return distill_t<T, 64, 16, true>(a, s);
    if (n <= 2048) return few ? distill_t<T, 256, 8, true>(a, s) : distill_t<T, 64, 32, true>(a, s);
    if (n <= 4096) return distill_t<T, 256, 16, true>(a, s);
    if (n <= 8192) return distill_t<T, 256, 32, false>(a, s);
    if (n <= 16384) return distill_t<T, 256, 64, false>(a, s);
    if (n <= 32768) return distill_t<T, 512, 64, false>(a, s);
    if constexpr (sizeof(T) == 2) {
        if (n <= 65536) return distill_t<T, 1024, 64, false>(a, s);
        return distill_t<T, 512, 192, false, true>(a, s);
    } else {
        if (n <= 65536) return distill_t<T, 512, 128, false>(a, s);
        return distill_t<T, 512, 96, false, true>(a, s);
    }
}

}  // namespace

hipError_t launch_distill(const DistillArgs &a, uint32_t dtype, hipStream_t s) {
    return dtype ? distill_n<half_t>(a, s) : distill_n<float>(a, s);
}

}  // namespace skl

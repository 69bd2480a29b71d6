// Distillation: a teacher's entries (a CSR matrix T x V) against rows of a student's dense logits.
//
//     z = x / t, q = softmax(z), p = softmax(v / t) over the row's entries (or exp(v)), P = sum p
//     loss = t^2 sum_i p_i (ln p_i - z[c_i] + lse z)
//     dx_j = g t (P q_j - sum of the p_i with c_i = j)
//
// No counterpart in the reference, whose CSR matrices are only multiplied (src/csrspmm.cpp:28-75).
//
// A row of logits belongs to one CTA, or to a cluster of up to eight where there are too few rows to fill the chip: each takes
// a run of columns, and the running maximum and sum of exp(z - max) of the parts meet in distributed shared memory.  The entries of
// the teacher are few and are read by every CTA of the row.
//
// Sums, maxima and the loss are fp32; everything is taken relative to the row's maximum, so that neither values of the type's
// lowest nor infinities in masked columns meet a product: exp((x - m) c) is 0 there.
#pragma once

#include <cooperative_groups.h>
#include <math_constants.h>

#include "common.cuh"
#include "score_types.cuh"

namespace csrspmm_b200 {

constexpr int kDistillMostCtas = 8;  // of a row: the largest cluster that every device runs
constexpr float kLowest = -3.402823466e38f;

struct DistillParams {
    int T, V, nnz;
    const void* x;
    long long ldx;
    const int* row_ptr;
    const int* col_idx;
    const float* values;
    float temperature, inv_t;
    int log_probs;
    float* loss;
    float4* stats;        // per row: max x, sum exp(z - max z), max v, sum exp((v - max v) / t)  (log_probs: 0, 1)
    const float* weight;  // per row, g above
    long long weight_stride;
    void* dx;
    long long ldd;
};

__device__ __forceinline__ float exp2_approx(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// A maximum and a sum of exponentials relative to it
struct MaxSum {
    float m, s;
};
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b, float c)
{
    const float m = fmaxf(a.m, b.m);
    return {m, a.s * exp2_approx((a.m - m) * c) + b.s * exp2_approx((b.m - m) * c)};
}

// What a thread sees of a row's part [c0, c1): whole 16-byte vectors from the first aligned element on, the rest one by one.
template <class T>
struct Part {
    static constexpr int N = 16 / (int)sizeof(T);
    int head, vectors, tail0;  // elements [c0, c0 + head), then `vectors` vectors, then [tail0, c1)
    __device__ __forceinline__ Part(const T* row, int c0, int c1)
    {
        const int off = (int)((reinterpret_cast<uintptr_t>(row + c0) & 15u) / sizeof(T));
        head = min(off ? N - off : 0, c1 - c0);
        vectors = (c1 - c0 - head) / N;
        tail0 = c0 + head + vectors * N;
    }
};

template <int THREADS>
struct BlockSums {
    float v[THREADS / 32];
};

// The sum over the block, in every thread; `room` is free again after the next barrier.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, BlockSums<THREADS>& room)
{
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) room.v[threadIdx.x >> 5] = v;
    __syncthreads();
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) sum += room.v[w];
    return sum;
}
template <int THREADS>
__device__ __forceinline__ float block_max(float v, BlockSums<THREADS>& room)
{
    v = warp_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) room.v[threadIdx.x >> 5] = v;
    __syncthreads();
    float m = room.v[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) m = fmaxf(m, room.v[w]);
    return m;
}

// The teacher's entries of a row
struct Teacher {
    int begin, count;
    const int* cols;
    const float* v;
    float top, sum;  // p = exp((v - top) / t) / sum

    __device__ __forceinline__ float share(const DistillParams& p, int i) const
    {
        const float at = __ldg(v + i);
        if (p.log_probs) return expf(at);
        return at > -CUDART_INF_F ? expf((at - top) * p.inv_t) / sum : at != at ? at : 0.0f;
    }
    __device__ __forceinline__ int column(const DistillParams& p, int i) const { return min(max(__ldg(cols + i), 0), p.V - 1); }
};

__device__ __forceinline__ Teacher teacher_of(const DistillParams& p, int row)
{
    Teacher t;
    t.begin = min(max(__ldg(p.row_ptr + row), 0), p.nnz);
    t.count = max(min(__ldg(p.row_ptr + row + 1), p.nnz) - t.begin, 0);
    t.cols = p.col_idx + t.begin;
    t.v = p.values + t.begin;
    t.top = 0.0f;
    t.sum = 1.0f;
    return t;
}

// The columns a CTA of the row takes.
__device__ __forceinline__ void part_bounds(int V, int part, int parts, int* c0, int* c1)
{
    const int per = ((V + parts - 1) / parts + 63) / 64 * 64;
    *c0 = (int)min((long long)part * per, (long long)V);
    *c1 = (int)min((long long)*c0 + per, (long long)V);
}

constexpr int kDistillUnroll = 4;  // vectors a thread has on their way

// Maximum and sum of exp((x - max) c / log2 e) over a part, per thread
template <class T, int THREADS>
__device__ __forceinline__ MaxSum scan_part(const T* row, int c0, int c1, float c)
{
    constexpr int N = Part<T>::N;
    const Part<T> part(row, c0, c1);
    MaxSum mine = {kLowest, 0.0f};
    const auto take = [&](const float* x, int n) {
        float top = x[0];
        for (int i = 1; i < n; ++i) top = fmaxf(top, x[i]);
        if (top > mine.m) {
            mine.s *= exp2_approx((mine.m - top) * c);
            mine.m = top;
        }
        for (int i = 0; i < n; ++i) mine.s += exp2_approx((x[i] - mine.m) * c);
    };
    const uint4* body = reinterpret_cast<const uint4*>(row + c0 + part.head);
    int at = threadIdx.x;
    for (; at + (kDistillUnroll - 1) * THREADS < part.vectors; at += kDistillUnroll * THREADS) {
        uint4 raw[kDistillUnroll];
#pragma unroll
        for (int u = 0; u < kDistillUnroll; ++u) raw[u] = __ldg(body + at + u * THREADS);
        float x[kDistillUnroll * N];
#pragma unroll
        for (int u = 0; u < kDistillUnroll; ++u) {
            const T* e = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
            for (int i = 0; i < N; ++i) x[u * N + i] = to_f32(e[i]);
        }
        float top = x[0];
#pragma unroll
        for (int i = 1; i < kDistillUnroll * N; ++i) top = fmaxf(top, x[i]);
        if (top > mine.m) {
            mine.s *= exp2_approx((mine.m - top) * c);
            mine.m = top;
        }
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kDistillUnroll * N; ++i) sum[i & 3] += exp2_approx((x[i] - mine.m) * c);
        mine.s += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
    for (; at < part.vectors; at += THREADS) {
        const uint4 raw = __ldg(body + at);
        const T* e = reinterpret_cast<const T*>(&raw);
        float x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = to_f32(e[i]);
        take(x, N);
    }
    for (int i = threadIdx.x; i < part.head; i += THREADS) {
        const float x = to_f32(row[c0 + i]);
        take(&x, 1);
    }
    for (int i = part.tail0 + threadIdx.x; i < c1; i += THREADS) {
        const float x = to_f32(row[i]);
        take(&x, 1);
    }
    return mine;
}

// dx over a part: first weight t P q everywhere, then the entries' columns again with their p taken off.
template <class T, int THREADS>
__device__ __forceinline__ void write_part(const DistillParams& p, const T* row, T* out, int c0, int c1, float c, float m, float s, const Teacher& t,
                                           float mass, float weight)
{
    constexpr int N = Part<T>::N;
    const float scale = weight * p.temperature * mass / s;
    const Part<T> part(row, c0, c1);
    const auto value = [&](T x) { return scale * exp2_approx((to_f32(x) - m) * c); };
    const uint4* body = reinterpret_cast<const uint4*>(row + c0 + part.head);
    T* to = out + c0 + part.head;
    const bool aligned = (reinterpret_cast<uintptr_t>(to) & 15u) == 0;
    for (int at = threadIdx.x; at < part.vectors; at += kDistillUnroll * THREADS) {
        uint4 raw[kDistillUnroll];
#pragma unroll
        for (int u = 0; u < kDistillUnroll; ++u)
            if (at + u * THREADS < part.vectors) raw[u] = __ldg(body + at + u * THREADS);
#pragma unroll
        for (int u = 0; u < kDistillUnroll; ++u) {
            const int k = at + u * THREADS;
            if (k < part.vectors) {
                const T* e = reinterpret_cast<const T*>(&raw[u]);
                Pack<T, N> r;
#pragma unroll
                for (int i = 0; i < N; ++i) r.v[i] = from_f32<T>(value(e[i]));
                if (aligned) {
                    *reinterpret_cast<Pack<T, N>*>(to + (long long)k * N) = r;
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) to[(long long)k * N + i] = r.v[i];
                }
            }
        }
    }
    for (int i = threadIdx.x; i < part.head; i += THREADS) out[c0 + i] = from_f32<T>(value(row[c0 + i]));
    for (int i = part.tail0 + threadIdx.x; i < c1; i += THREADS) out[i] = from_f32<T>(value(row[i]));
    // A column that is named more than once is written by its first entry, with all its p in stored order.  Ascending columns
    // name none twice.
    bool ascending = true;
    for (int i = threadIdx.x; i + 1 < t.count; i += THREADS) ascending &= t.column(p, i) < t.column(p, i + 1);
    const bool distinct = __syncthreads_and(ascending);  // and the rows' writes above come before those below
    for (int i = threadIdx.x; i < t.count; i += THREADS) {
        const int col = t.column(p, i);
        if (col < c0 || col >= c1) continue;
        float share = t.share(p, i);
        if (!distinct) {
            bool first = true;
            for (int j = 0; j < i && first; ++j) first = t.column(p, j) != col;
            if (!first) continue;
            for (int j = i + 1; j < t.count; ++j)
                if (t.column(p, j) == col) share += t.share(p, j);
        }
        out[col] = from_f32<T>(weight * p.temperature * (mass * (exp2_approx((to_f32(row[col]) - m) * c) / s) - share));
    }
}

template <class T, int THREADS>
__device__ __forceinline__ void zero_part(T* out, int c0, int c1)
{
    constexpr int N = Part<T>::N;
    const Part<T> part(out, c0, c1);
    for (int at = threadIdx.x; at < part.vectors; at += THREADS) *reinterpret_cast<uint4*>(out + c0 + part.head + (long long)at * N) = make_uint4(0, 0, 0, 0);
    for (int i = threadIdx.x; i < part.head; i += THREADS) out[c0 + i] = from_f32<T>(0.0f);
    for (int i = part.tail0 + threadIdx.x; i < c1; i += THREADS) out[i] = from_f32<T>(0.0f);
}

// The loss of a row, and with GRADIENT its dx in the same launch.  Grid: T rows of gridDim.x / T CTAs, a cluster each where that is more than one.
template <class T, int THREADS, bool GRADIENT, bool CLUSTER>
__global__ void __launch_bounds__(THREADS) distill_kernel(DistillParams p)
{
    namespace cg = cooperative_groups;
    __shared__ BlockSums<THREADS> room;
    __shared__ MaxSum of_warp[THREADS / 32];
    __shared__ MaxSum of_block;
    wait_for_previous_grid();
    const int parts = CLUSTER ? (int)cg::this_cluster().num_blocks() : 1;
    const int rank = CLUSTER ? (int)cg::this_cluster().block_rank() : 0;
    const int row = (int)(blockIdx.x / parts);
    int c0, c1;
    part_bounds(p.V, rank, parts, &c0, &c1);
    const T* x = static_cast<const T*>(p.x) + (long long)row * p.ldx;
    const float c = p.inv_t * CUDART_L2E_F;
    Teacher t = teacher_of(p, row);

    if (!p.log_probs) {
        float top = -CUDART_INF_F;
        bool broken = false;
        for (int i = threadIdx.x; i < t.count; i += THREADS) {
            const float v = __ldg(t.v + i);
            top = fmaxf(top, v);
            broken |= v != v;
        }
        t.top = block_max<THREADS>(top, room);
        if (__syncthreads_or(broken)) t.top = CUDART_NAN_F;
        if (t.top == -CUDART_INF_F) t.count = 0;  // no entry, or none that weighs anything
    }
    if (t.count == 0) {  // every CTA of the row leaves here
        if (rank == 0 && threadIdx.x == 0) {
            p.loss[row] = 0.0f;
            if (p.stats != nullptr) p.stats[row] = make_float4(0.0f, 1.0f, -CUDART_INF_F, 1.0f);
        }
        if constexpr (GRADIENT) zero_part<T, THREADS>(static_cast<T*>(p.dx) + (long long)row * p.ldd, c0, c1);
        return;
    }

    MaxSum mine = scan_part<T, THREADS>(x, c0, c1, c);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
        const MaxSum other = {__shfl_xor_sync(kAllLanes, mine.m, d), __shfl_xor_sync(kAllLanes, mine.s, d)};
        mine = join(mine, other, c);
    }
    if ((threadIdx.x & 31) == 0) of_warp[threadIdx.x >> 5] = mine;
    __syncthreads();
    mine = of_warp[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) mine = join(mine, of_warp[w], c);
    if constexpr (CLUSTER) {
        const cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x == 0) of_block = mine;
        cluster.sync();
        mine = *cluster.map_shared_rank(&of_block, 0);
        for (int r = 1; r < parts; ++r) mine = join(mine, *cluster.map_shared_rank(&of_block, r), c);
        cluster.sync();  // nobody leaves while another reads
    }

    // with e = exp((v - top) / t): sum e, and sum e ((v - top) / t - (z - max z))
    float sum = 0.0f, cross = 0.0f;
    for (int i = threadIdx.x; i < t.count; i += THREADS) {
        const float v = __ldg(t.v + i);
        const float over = p.log_probs ? v : (v - t.top) * p.inv_t;
        const float e = expf(over);
        sum += e;
        if (e != 0.0f && rank == 0) cross += e * (over - (to_f32(x[t.column(p, i)]) - mine.m) * p.inv_t);
    }
    sum = block_sum<THREADS>(sum, room);
    if (!p.log_probs) t.sum = sum;
    const float mass = p.log_probs || sum != sum ? sum : 1.0f;
    if (rank == 0) {
        cross = block_sum<THREADS>(cross, room);
        if (threadIdx.x == 0) {
            const float lse = logf(mine.s);
            p.loss[row] = mass == 0.0f ? 0.0f : p.temperature * p.temperature * (p.log_probs ? cross + mass * lse : cross / sum - logf(sum) + lse);
            if (p.stats != nullptr) p.stats[row] = make_float4(mine.m, mine.s, t.top, sum);
        }
    }
    if constexpr (GRADIENT) {
        T* out = static_cast<T*>(p.dx) + (long long)row * p.ldd;
        if (mass == 0.0f) zero_part<T, THREADS>(out, c0, c1);
        else write_part<T, THREADS>(p, x, out, c0, c1, c, mine.m, mine.s, t, mass, __ldg(p.weight + row * p.weight_stride));
    }
}

// dx from the statistics that the loss left.  Grid: T rows of gridDim.x / T CTAs.
template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS) distill_backward_kernel(DistillParams p, int parts)
{
    wait_for_previous_grid();
    const int row = (int)(blockIdx.x / parts);
    int c0, c1;
    part_bounds(p.V, (int)(blockIdx.x % parts), parts, &c0, &c1);
    const T* x = static_cast<const T*>(p.x) + (long long)row * p.ldx;
    T* out = static_cast<T*>(p.dx) + (long long)row * p.ldd;
    Teacher t = teacher_of(p, row);
    const float4 stats = __ldg(p.stats + row);
    t.top = stats.z;
    t.sum = p.log_probs ? 1.0f : stats.w;
    const float mass = p.log_probs || stats.w != stats.w ? stats.w : 1.0f;
    if (t.count == 0 || stats.z == -CUDART_INF_F || mass == 0.0f) zero_part<T, THREADS>(out, c0, c1);
    else write_part<T, THREADS>(p, x, out, c0, c1, p.inv_t * CUDART_L2E_F, stats.x, stats.y, t, mass, __ldg(p.weight + row * p.weight_stride));
}

}  // namespace csrspmm_b200

// Distillation: a teacher's entries (a CSR matrix T x V) against rows of a student's dense logits.
//
//     z = x / t, q = softmax(z), p = softmax(v / t) over the row's entries (or exp(v)), P = sum p
//     loss = t^2 sum_i p_i (ln p_i - z[c_i] + lse z)
//     dx_j = g t (P q_j - sum of the p_i with c_i = j)
//
// No counterpart in the reference, whose CSR matrices are only multiplied (src/csrspmm.cpp:28-75).
//
// Loss, and loss with gradient (distill_ring_kernel): a row of logits belongs to a CTA or to a cluster of up to eight, each of which takes a
// run of columns.  Bulk copies bring the run into shared memory and the runs of the next rows behind it, so that memory is never waited for row by
// row; from there it is read for the maximum, for the sum and for the gradient, and memory gives each row once.  What
// the parts found meets in distributed shared memory.  The teacher's entries are few: one warp makes their shares.
// The gradient alone (distill_gradient_kernel) needs no sum: every thread holds up to eight vectors.  Rows that one warp can hold are a
// warp's (distill_short_kernel); rows that are longer than a cluster's shared memory are read twice (distill_long_kernel).
//
// Sums, maxima and the loss are fp32.  Exponentials are 2^y with y = x c - m c, c = log2(e) / t, m a maximum: one fused multiply-add each.  The
// product m c is rounded once and the same rounded one serves the sum, the loss and the gradient, so that its rounding cancels.  That holds
// while its rounding is small as an exponent: from |m c| = 2^24 on, where it passes a half (a row of a mask such as -1e30; beyond 2^31 it alone
// would overflow 2^y), y = (x - m) c.
#pragma once

#include <cooperative_groups.h>
#include <math_constants.h>

#include <type_traits>

#include "async_copy.cuh"
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
    float4* stats;        // per row: max x, sum exp(z - max z), max v, sum exp((v - max v) / t)  (log_probs: 0, sum exp v)
    const float* weight;  // per row, g above
    long long weight_stride;
    void* dx;
    long long ldd;
    int log_parts, per;  // a row is cut into 2^log_parts runs of `per` columns, a multiple of 64
    // the ring kernel's: rows of a CTA or cluster, copies on their way and the room of each, the shared memory before them
    int rows, slots, slot_bytes, ring_offset;
    unsigned wait_limit;  // attempts of a wait for a copy
};

__device__ __forceinline__ float exp2_approx(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

__device__ __forceinline__ Pair exp2_approx(Pair v)
{
    const float2 w = halves(v);
    return pair_of(exp2_approx(w.x), exp2_approx(w.y));
}

constexpr float kFarProduct = 16777216.0f;  // 2^24: below it a product is off by at most a half

// y above, for one maximum
struct Exponent {
    float m, mc, c;
    bool far;
    __device__ __forceinline__ Exponent(float top, float scale)
    {
        m = top;
        c = scale;
        mc = __fmul_rn(top, scale);
        far = !(fabsf(mc) < kFarProduct);
    }
    template <bool FAR>
    __device__ __forceinline__ float of(float x) const
    {
        return FAR ? (x - m) * c : __fmaf_rn(x, c, -mc);
    }
    __device__ __forceinline__ float of(float x) const { return far ? of<true>(x) : of<false>(x); }
    template <bool FAR>
    __device__ __forceinline__ Pair of(Pair x) const
    {
        if constexpr (FAR) {
            const float2 v = halves(x);
            return pair_of(of<true>(v.x), of<true>(v.y));
        } else {
            return fma2(x, pair_of(c, c), pair_of(-mc, -mc));
        }
    }
    // what y is too large by: the rounding of m c
    __device__ __forceinline__ float excess() const { return far ? 0.0f : __fmaf_rn(m, c, -mc); }
    // of a smaller maximum, to which its own sum was taken: with the rounding of its product too, or without where that one is far
    __device__ __forceinline__ float of_max(float other) const
    {
        const Exponent o(other, c);
        const float apart = (other - m) * c + (excess() - o.excess());  // without a branch: lanes that hold nothing are far
        return far || o.far ? apart : __fsub_rn(o.mc, mc);
    }
    // (x - m) / t for the loss, where x log2(e) / t may pass fp32 while x / t does not: a teacher's entry where the student holds the type's lowest
    __device__ __forceinline__ float below(float x, float inv_t) const { return natural(of(x), x, inv_t); }
    __device__ __forceinline__ float max_below(float other, float inv_t) const { return natural(of_max(other), other, inv_t); }
    __device__ __forceinline__ float natural(float y, float x, float inv_t) const
    {
        return fabsf(y) <= -kLowest ? y * CUDART_LN2_F : x * inv_t - m * inv_t;
    }
};

// The entries' sum of e (v / t - (z - max z)) is kept in this unit where e is relative to the largest: a few e of 1 times the type's lowest pass fp32
// before they are divided by the sum of the e.  (With log_probs the e are the p themselves.)
constexpr float kCrossUnit = 5.9604644775390625e-8f, kPerCrossUnit = 16777216.0f;  // 2^-24
__device__ __forceinline__ float cross_unit(const DistillParams& p) { return p.log_probs ? 1.0f : kCrossUnit; }
// A row's loss but for t^2; sum: sum e, mass: P, lse: the logarithm of the sum of exp(z - max z)
__device__ __forceinline__ float divergence(const DistillParams& p, float cross, float sum, float mass, float lse)
{
    return p.log_probs ? cross + mass * lse : cross / sum * kPerCrossUnit - logf(sum) + lse;
}

// A maximum and the sum of 2^y relative to it; none: kLowest and 0.
struct MaxSum {
    float m, s;
};
// What a thread sees of a row's part [c0, c1): whole 16-byte vectors from the first aligned element on; of the at most
// 2 (N - 1) elements before and behind, one a thread.
template <class T>
struct Part {
    static constexpr int N = 16 / (int)sizeof(T);
    int first, vectors, edge;  // the first vector's column; this thread's single element, or -1
    __device__ __forceinline__ Part(const T* row, int c0, int c1)
    {
        const int off = (int)((reinterpret_cast<uintptr_t>(row + c0) & 15u) / sizeof(T));
        const int head = min(off ? N - off : 0, c1 - c0);
        first = c0 + head;
        vectors = (c1 - first) / N;
        const int behind = first + vectors * N, tid = (int)threadIdx.x;
        edge = tid < head ? c0 + tid : behind + (tid - head) < c1 ? behind + (tid - head) : -1;
    }
};

// The row and the columns that a CTA takes.
struct Place {
    int row, rank, c0, c1;
    __device__ __forceinline__ explicit Place(const DistillParams& p) : Place(p, (int)(blockIdx.x >> p.log_parts)) {}
    __device__ __forceinline__ Place(const DistillParams& p, int r)
    {
        row = r;
        rank = (int)blockIdx.x & ((1 << p.log_parts) - 1);
        c0 = (int)min((long long)rank * p.per, (long long)p.V);
        c1 = (int)min((long long)c0 + p.per, (long long)p.V);
    }
};

// The teacher's entries of a row
struct Teacher {
    int count;
    const int* cols;
    const float* v;
    float top, sum;  // p = exp((v - top) / t) / sum

    __device__ __forceinline__ float share(const DistillParams& p, float at) const
    {
        if (p.log_probs) return expf(at);
        return at > -CUDART_INF_F ? expf((at - top) * p.inv_t) / sum : at != at ? at : 0.0f;
    }
    __device__ __forceinline__ int column(const DistillParams& p, int i) const { return min(max(__ldg(cols + i), 0), p.V - 1); }
};

__device__ __forceinline__ Teacher teacher_of(const DistillParams& p, int from, int to)  // its two row offsets
{
    Teacher t;
    const int begin = min(max(from, 0), p.nnz);
    t.count = max(min(to, p.nnz) - begin, 0);
    t.cols = p.col_idx + begin;
    t.v = p.values + begin;
    t.top = 0.0f;
    t.sum = 1.0f;
    return t;
}

// An entry, and the student's logit in its column
struct Entry {
    float v, x;
    int col;
};

// A thread's entries: the first is asked for at once and used late.
template <class T, int THREADS>
struct Entries {
    const DistillParams& p;
    const Teacher& t;
    const T* row;
    Entry first = {};
    __device__ __forceinline__ Entries(const DistillParams& params, const Teacher& teacher, const T* x) : p(params), t(teacher), row(x)
    {
        if ((int)threadIdx.x < t.count) first = load(threadIdx.x);
    }
    __device__ __forceinline__ Entry load(int i) const
    {
        Entry e;
        e.col = t.column(p, i);
        e.v = __ldg(t.v + i);
        e.x = to_f32(row[e.col]);
        return e;
    }
    template <class F>
    __device__ __forceinline__ void each(F&& f) const
    {
        if ((int)threadIdx.x < t.count) f((int)threadIdx.x, first);
        for (int i = threadIdx.x + THREADS; i < t.count; i += THREADS) f(i, load(i));
    }
};

// What the warps of a CTA hand one another
template <int THREADS>
struct Room {
    MaxSum part[THREADS / 32];
    float top[THREADS / 32], sum[THREADS / 32], cross[THREADS / 32];
    MaxSum block;
};

// The maximum and sum of N lanes' (a power of two), each its own: the largest maximum first, then every sum is brought to it once.
template <int N>
__device__ __forceinline__ MaxSum join_lanes(MaxSum mine, float c)
{
    float m = mine.m;
#pragma unroll
    for (int d = N / 2; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(kAllLanes, m, d));
    float s = mine.s * exp2_approx(Exponent(m, c).of_max(mine.m));
#pragma unroll
    for (int d = N / 2; d > 0; d >>= 1) s += __shfl_xor_sync(kAllLanes, s, d);
    return {m, s};
}

// Maximum and sum of the row from the warps' (with the other CTAs' of its cluster), in every thread; ends the first of the phases that
// a barrier parts.
template <int THREADS>
__device__ __forceinline__ MaxSum join_row(MaxSum warps, float c, Room<THREADS>& room, int log_parts)
{
    namespace cg = cooperative_groups;
    constexpr int W = THREADS / 32;
    const int lane = threadIdx.x & 31;
    if (lane == 0) room.part[threadIdx.x >> 5] = warps;
    __syncthreads();
    MaxSum all = join_lanes<W>(room.part[lane % W], c);
    if (log_parts > 0) {
        const cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x == 0) room.block = all;
        cluster.sync();
        const int parts = 1 << log_parts;
        all = join_lanes<8>(lane % 8 < parts ? *cluster.map_shared_rank(&room.block, lane % 8) : MaxSum{kLowest, 0.0f}, c);
    }
    return all;
}
// Nobody leaves while another may still read what it left in join_row.
__device__ __forceinline__ void leave_row(int log_parts)
{
    if (log_parts > 0) cooperative_groups::this_cluster().sync();
}

// The largest of the entries' values (NaN where one is), of the warps that have any; read after join_row's barrier.
template <class T, int THREADS>
__device__ __forceinline__ void leave_top(const Entries<T, THREADS>& entries, Room<THREADS>& room)
{
    const int warp = threadIdx.x >> 5;
    float top = -CUDART_INF_F;
    if (warp * 32 < entries.t.count) {
        bool broken = false;
        entries.each([&](int, const Entry& e) {
            top = fmaxf(top, e.v);
            broken |= e.v != e.v;
        });
        top = warp_max(top);
        if (__any_sync(kAllLanes, broken)) top = CUDART_NAN_F;
    }
    if ((threadIdx.x & 31) == 0) room.top[warp] = top;
}
template <int THREADS>
__device__ __forceinline__ float joined_top(const Room<THREADS>& room)
{
    constexpr int W = THREADS / 32;
    const float top = room.top[(threadIdx.x & 31) % W];
    return __any_sync(kAllLanes, top != top) ? CUDART_NAN_F : warp_max(top);
}

// The entries' sums, and the row's loss by the first CTA of the row.  Returns P; t.sum is set after it.
template <class T, int THREADS>
__device__ __forceinline__ float finish_loss(const DistillParams& p, const Place& at, const Entries<T, THREADS>& entries, Teacher& t, const Exponent& y,
                                             float s, Room<THREADS>& room)
{
    constexpr int W = THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // with e = exp((v - top) / t): sum e, and sum e ((v - top) / t - (z - max z))
    const float unit = cross_unit(p);
    float sum = 0.0f, cross = 0.0f;
    if (warp * 32 < t.count) {
        entries.each([&](int, const Entry& e) {
            const float over = p.log_probs ? e.v : (e.v - t.top) * p.inv_t;
            const float share = expf(over);
            sum += share;
            if (share != 0.0f) cross += share * ((over - y.below(e.x, p.inv_t)) * unit);
        });
        sum = warp_sum(sum);
        cross = warp_sum(cross);
    }
    if (lane == 0) room.sum[warp] = sum, room.cross[warp] = cross;
    __syncthreads();
    sum = room.sum[lane % W];
#pragma unroll
    for (int d = W / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(kAllLanes, sum, d);
    if (!p.log_probs) t.sum = sum;
    const float mass = p.log_probs || sum != sum ? sum : 1.0f;
    if (at.rank == 0 && warp == 0) {
        cross = warp_sum(lane < W ? room.cross[lane] : 0.0f);
        if (lane == 0) {
            const float lse = logf(s), tt = p.temperature * p.temperature;
            p.loss[at.row] = mass == 0.0f ? 0.0f : tt * divergence(p, cross, sum, mass, lse);
            if (p.stats != nullptr) p.stats[at.row] = make_float4(y.m, s, t.top, sum);
        }
    }
    return mass;
}

template <class T, int THREADS>
__device__ __forceinline__ void zero_part(T* out, int c0, int c1)
{
    const Part<T> part(out, c0, c1);
    for (int at = threadIdx.x; at < part.vectors; at += THREADS) *reinterpret_cast<uint4*>(out + part.first + (long long)at * Part<T>::N) = make_uint4(0, 0, 0, 0);
    if (part.edge >= 0) out[part.edge] = from_f32<T>(0.0f);
}

// A row without a teacher: every CTA of it leaves here.
template <class T, int THREADS>
__device__ __forceinline__ void leave_out(const DistillParams& p, const Place& at, bool loss, bool gradient)
{
    if (loss && at.rank == 0 && threadIdx.x == 0) {
        p.loss[at.row] = 0.0f;
        if (p.stats != nullptr) p.stats[at.row] = make_float4(0.0f, 1.0f, -CUDART_INF_F, 1.0f);
    }
    if (gradient) zero_part<T, THREADS>(static_cast<T*>(p.dx) + (long long)at.row * p.ldd, at.c0, at.c1);
}

// A vector of dx at `to`, which need not be aligned
template <class T>
__device__ __forceinline__ void store_vector(T* to, const uint4& v, bool aligned)
{
    if (aligned) {
        *reinterpret_cast<uint4*>(to) = v;
    } else {
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int i = 0; i < Part<T>::N; ++i) to[i] = e[i];
    }
}

// What becomes of the columns of a row's entries where some may be named more than once: each is written with all its p.
template <class T>
struct NamedColumns {
    float* sums;  // `span` floats of a warp's own
    int span, part, parts;  // this warp's place among those that share the work
    int c0, c1, V;          // columns that are written
    Teacher t;
    int log_probs;
    float inv_t, c, m;       // of the exponentials
    float scale, taken;      // dx = scale 2^y - taken * sum p
    const T* x;
    T* out;
};

// One warp's part: it walks over the entries once for every `span` columns and adds up their p in a fixed order, in time that grows with the entries
// where comparing them with one another takes their square.
template <class T, int U>  // U columns a lane on their way at once
__device__ __forceinline__ void write_named_columns(NamedColumns<T> a)
{
    const int lane = threadIdx.x & 31;
    const Exponent y(a.m, a.c);
    for (long long base = a.c0 + (long long)a.part * a.span; base < a.c1; base += (long long)a.parts * a.span) {
        const int from = (int)base, width = min(a.span, a.c1 - from);
        for (int k = lane; k < width; k += 32) a.sums[k] = -1.0f;  // named by none
        __syncwarp();
        for (long long j0 = lane; j0 - lane < a.t.count; j0 += 32 * U) {
            int at[U];
#pragma unroll
            for (int u = 0; u < U; ++u) at[u] = j0 + u * 32 < a.t.count ? min(max(__ldg(a.t.cols + j0 + u * 32), 0), a.V - 1) - from : -1;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const bool mine = at[u] >= 0 && at[u] < width;
                if (!__any_sync(kAllLanes, mine)) continue;
                float p = 0.0f;
                if (mine) {
                    const float v = __ldg(a.t.v + j0 + u * 32);
                    p = a.log_probs ? expf(v) : v > -CUDART_INF_F ? expf((v - a.t.top) * a.inv_t) / a.t.sum : v != v ? v : 0.0f;
                }
                const unsigned same = __match_any_sync(kAllLanes, mine ? at[u] : -1 - lane);
                if (__any_sync(kAllLanes, (same & (same - 1)) != 0)) {  // lanes of one column: each adds what follows it, by steps that double
                    const unsigned above = same & ~((2u << lane) - 1u);
                    int next = above != 0 ? __ffs(above) - 1 : -1;
#pragma unroll
                    for (int d = 0; d < 5; ++d) {
                        const float v = __shfl_sync(kAllLanes, p, next & 31);
                        const int n = __shfl_sync(kAllLanes, next, next & 31);
                        if (next >= 0) p += v, next = n;
                    }
                }
                if (mine && __ffs(same) - 1 == lane) a.sums[at[u]] = a.sums[at[u]] < 0.0f ? p : a.sums[at[u]] + p;
                __syncwarp();
            }
        }
        for (int k = lane; k < width; k += 32)
            if (!(a.sums[k] < 0.0f)) a.out[from + k] = from_f32<T>(a.scale * exp2_approx(y.of(to_f32(a.x[from + k]))) - a.taken * a.sums[k]);
        __syncwarp();
    }
}

// The columns of the entries again, over what was written there: their p taken off.  `repeats`: a column may be named more than once; `sums`: `span`
// floats for each warp.
template <class T, int THREADS>
__device__ __forceinline__ void write_entries(const DistillParams& p, const Entries<T, THREADS>& entries, const Teacher& t, const Exponent& y, float scale,
                                              float weight, T* out, int c0, int c1, bool repeats, float* sums, int span)
{
    if (repeats) {
        const int warp = threadIdx.x >> 5;
        write_named_columns<T, 4>({sums + warp * span, span, warp, THREADS / 32, c0, c1, p.V, t, p.log_probs, p.inv_t, y.c, y.m, scale,
                                   weight * p.temperature, entries.row, out});
    } else {
        entries.each([&](int, const Entry& e) {
            if (e.col >= c0 && e.col < c1) out[e.col] = from_f32<T>(scale * exp2_approx(y.of(e.x)) - weight * p.temperature * t.share(p, e.v));
        });
    }
}

// dx from the statistics that the loss left.  Grid: T rows of 2^log_parts CTAs.  A part has at most THREADS * NV vectors, all of which are
// asked for before anything else; two CTAs of 512 threads, or as many smaller ones, share an SM.
template <class T, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) distill_gradient_kernel(DistillParams p)
{
    constexpr int N = Part<T>::N;
    constexpr int kNamedWords = THREADS * NV * N / 32 + 2;  // the part's vectors, and what is before and behind them
    constexpr int kSpan = 128;                              // for a warp's sums: at most 16 walks over the entries
    __shared__ union {
        unsigned named[kNamedWords];  // a bit for each column of the part
        float sums[THREADS / 32 * kSpan];
    } sh;
    wait_for_previous_grid();
    const Place at(p);
    const T* x = static_cast<const T*>(p.x) + (long long)at.row * p.ldx;
    const Part<T> part(x, at.c0, at.c1);
    uint4 held[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (int)threadIdx.x + i * THREADS;
        if (k < part.vectors) held[i] = load_once(x + part.first + k * N);
    }
    const float edge = part.edge >= 0 ? to_f32(x[part.edge]) : 0.0f;
    const float4 stats = __ldg(p.stats + at.row);
    Teacher t = teacher_of(p, __ldg(p.row_ptr + at.row), __ldg(p.row_ptr + at.row + 1));
    t.top = stats.z;
    t.sum = p.log_probs ? 1.0f : stats.w;
    const float mass = p.log_probs || stats.w != stats.w ? stats.w : 1.0f;
    if (t.count == 0 || stats.z == -CUDART_INF_F || mass == 0.0f) {
        leave_out<T, THREADS>(p, at, false, true);
        return;
    }
    const Entries<T, THREADS> entries(p, t, x);
    for (int i = threadIdx.x; i < kNamedWords; i += THREADS) sh.named[i] = 0;
    const float c = p.inv_t * CUDART_L2E_F;
    const Exponent y(stats.x, c);
    const float weight = __ldg(p.weight + at.row * p.weight_stride);
    const float scale = weight * p.temperature * mass / stats.y;
    T* out = static_cast<T*>(p.dx) + (long long)at.row * p.ldd;
    T* to = out + part.first;
    const bool aligned = (reinterpret_cast<uintptr_t>(to) & 15u) == 0;
    __syncthreads();
    const auto write = [&](auto far) {
        const auto value = [&](Pair v) { return mul2(pair_of(scale, scale), exp2_approx(y.template of<decltype(far)::value>(v))); };
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = (int)threadIdx.x + i * THREADS;
            if (k < part.vectors) store_vector(to + k * N, Words<T>::map(held[i], value), aligned);
        }
        if (part.edge >= 0) out[part.edge] = from_f32<T>(scale * exp2_approx(y.of(edge)));
    };
    if (y.far) write(std::true_type());
    else write(std::false_type());
    bool repeats = false;
    const bool named_here = (int)(threadIdx.x & ~31u) < t.count;
    if (named_here) {
        entries.each([&](int, const Entry& e) {
            const int k = e.col - at.c0;
            if (k >= 0 && k < at.c1 - at.c0) repeats |= (atomicOr(&sh.named[k >> 5], 1u << (k & 31)) >> (k & 31)) & 1u;
        });
    }
    repeats = __syncthreads_or(repeats);  // and what was written above comes before what is written below
    if (named_here || repeats) write_entries<T, THREADS>(p, entries, t, y, scale, weight, out, at.c0, at.c1, repeats, sh.sums, kSpan);
}

// Short rows: a warp each, which holds its row in registers, up to NV vectors a lane.  (Under the ring's two warps of a CTA a row of 1500 bf16
// logits took 15 us from end to end, which 14 CTAs per SM do not hide: 16384 of them 122 us.)
constexpr int kShortThreads = 256;

template <class T, int NV, bool GRADIENT>
__global__ void __launch_bounds__(kShortThreads) distill_short_kernel(DistillParams p)
{
    constexpr int N = Part<T>::N, kSpan = 256;
    static_assert(kSpan * 32 >= 32 * NV * N, "a bit for each column of a row");
    __shared__ union {
        unsigned named[kSpan];
        float sums[kSpan];
    } of_warp[GRADIENT ? kShortThreads / 32 : 1];
    wait_for_previous_grid();
    const int lane = threadIdx.x & 31;
    const int row = (int)(blockIdx.x * (kShortThreads / 32) + (threadIdx.x >> 5));
    if (row >= p.T) return;
    const T* const x = static_cast<const T*>(p.x) + (long long)row * p.ldx;
    const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
    const int head = min(off ? N - off : 0, p.V), vectors = (p.V - head) / N, behind = head + vectors * N + lane - head;
    const int edge_col = lane < head ? lane : behind < p.V ? behind : -1;  // fewer than 2 N, a lane each
    uint4 held[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        constexpr unsigned none = Words<T>::kMinusInf;
        held[i] = lane + i * 32 < vectors ? load_once(x + head + (lane + i * 32) * N) : make_uint4(none, none, none, none);
    }
    const float edge = edge_col >= 0 ? to_f32(x[edge_col]) : -CUDART_INF_F;
    Teacher t = teacher_of(p, __ldg(p.row_ptr + row), __ldg(p.row_ptr + row + 1));
    const auto entry = [&](int j) {
        Entry e;
        e.col = t.column(p, j);
        e.v = __ldg(t.v + j);
        e.x = to_f32(x[e.col]);
        return e;
    };
    Entry first = {};
    if (lane < t.count) first = entry(lane);
    const auto each = [&](auto&& f) {
        if (lane < t.count) f(lane, first);
        for (int j = lane + 32; j < t.count; j += 32) f(j, entry(j));
    };

    const float c = p.inv_t * CUDART_L2E_F;
    unsigned top_words = Words<T>::kMinusInf;
#pragma unroll
    for (int i = 0; i < NV; ++i) top_words = max_words<T>(top_words, held[i]);
    const Exponent y(fmaxf(warp_max(fmaxf(Words<T>::largest(top_words), edge)), kLowest), c);
    Pair sum = pair_of(0.0f, 0.0f);
    const auto add = [&](auto far) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (i * 32 < vectors) Words<T>::each(held[i], [&](Pair w) { sum = add2(sum, exp2_approx(y.template of<decltype(far)::value>(w))); });
    };
    if (y.far) add(std::true_type());
    else add(std::false_type());
    const float s = warp_sum(halves(sum).x + halves(sum).y + exp2_approx(y.of(edge)));

    t.top = -CUDART_INF_F;
    t.sum = 0.0f;
    if (p.log_probs) {
        if (t.count > 0) t.top = 0.0f;
    } else {
        bool broken = false;
        each([&](int, const Entry& e) {
            t.top = fmaxf(t.top, e.v);
            broken |= e.v != e.v;
        });
        t.top = __any_sync(kAllLanes, broken) ? CUDART_NAN_F : warp_max(t.top);
    }
    const bool counts = t.top != -CUDART_INF_F;  // some entry weighs something
    const auto over_of = [&](float v) { return p.log_probs ? v : (v - t.top) * p.inv_t; };
    const float unit = cross_unit(p);
    float cross = 0.0f;
    if (counts) {
        each([&](int, const Entry& e) {
            const float over = over_of(e.v), share = expf(over);
            t.sum += share;
            if (share != 0.0f) cross += share * ((over - y.below(e.x, p.inv_t)) * unit);
        });
        t.sum = warp_sum(t.sum);
        cross = warp_sum(cross);
    }
    const float mass = !counts ? 0.0f : p.log_probs || t.sum != t.sum ? t.sum : 1.0f;
    const bool zero = mass == 0.0f;
    if (lane == 0) {
        const float lse = logf(s), tt = p.temperature * p.temperature;
        p.loss[row] = zero ? 0.0f : tt * divergence(p, cross, t.sum, mass, lse);
        if (p.stats != nullptr) p.stats[row] = counts ? make_float4(y.m, s, t.top, t.sum) : make_float4(0.0f, 1.0f, -CUDART_INF_F, 1.0f);
    }
    if constexpr (GRADIENT) {
        T* const out = static_cast<T*>(p.dx) + (long long)row * p.ldd;
        T* const to = out + head;
        const bool aligned = (reinterpret_cast<uintptr_t>(to) & 15u) == 0;
        const float weight = __ldg(p.weight + row * p.weight_stride), scale = weight * p.temperature * mass / s;
        const auto write = [&](auto far) {
            const auto value = [&](Pair v) { return mul2(pair_of(scale, scale), exp2_approx(y.template of<decltype(far)::value>(v))); };
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (lane + i * 32 < vectors) store_vector(to + (lane + i * 32) * N, zero ? make_uint4(0, 0, 0, 0) : Words<T>::map(held[i], value), aligned);
        };
        if (y.far) write(std::true_type());
        else write(std::false_type());
        if (edge_col >= 0) out[edge_col] = from_f32<T>(zero ? 0.0f : scale * exp2_approx(y.of(edge)));
        if (zero) return;
        bool repeats = false;
        auto& sh = of_warp[threadIdx.x >> 5];
        if (t.count <= 32) {
            const unsigned same = __match_any_sync(kAllLanes, lane < t.count ? first.col : -1 - lane);
            repeats = (same & (same - 1)) != 0;
        } else {
            for (int k = lane; k * 32 < p.V; k += 32) sh.named[k] = 0;
            __syncwarp();
            each([&](int, const Entry& e) { repeats |= (atomicOr(&sh.named[e.col >> 5], 1u << (e.col & 31)) >> (e.col & 31)) & 1u; });
        }
        repeats = __any_sync(kAllLanes, repeats);
        __syncwarp();  // what was written above comes before what is written below
        const auto share_of = [&](float v) { return p.log_probs ? expf(v) : expf(over_of(v)) / t.sum; };
        if (repeats) {
            write_named_columns<T, 2>({sh.sums, kSpan, 0, 1, 0, p.V, p.V, t, p.log_probs, p.inv_t, c, y.m, scale, weight * p.temperature, x, out});
        } else {
            each([&](int, const Entry& e) { out[e.col] = from_f32<T>(scale * exp2_approx(y.of(e.x)) - weight * p.temperature * share_of(e.v)); });
        }
    }
}

// ---- the ring ------------------------------------------------------------------------------------------
//
// WORKERS threads do what is done for every element and one more warp, the manager, all the rest: it starts the copies, makes the teacher's
// shares, joins maxima and sums (across the cluster too), writes the loss and the entries' columns.  What a row costs beside its elements
// is then paid by one warp in nine: when all warps took part, that was 600 of 1300 instructions of each, and the kernel was no
// faster than two plain sweeps (227 us for 1184 rows of 131072 bf16 logits).

constexpr int kListed = 256;  // entries of a row that are kept in shared memory; rows with more read them where they need them
constexpr int kMostSlots = 2;
constexpr int kMostRows = 4;  // of a CTA or cluster
// How much longer than a copy takes may be waited for what a manager does first, who may still walk over the entries of the row before.
constexpr unsigned kWalkFactor = 64;
constexpr unsigned kToldLimit = kWalkFactor * kWaitSpinLimit;

// From so many entries on the walk that writes the entries' columns comes after all rows, with the logits from memory, as it does where columns are
// named twice in more than a list: the workers wait for a copy, not for the walk.
constexpr int kLongWalk = 2048;

struct RingRow {  // what the workers need to write a part of dx
    float m, scale;
    int zero, aligned, vectors;
    void* to;
};

struct RingBlock {  // what a part hands to the others: its maximum and sum, and over its entries sum e (v / t - (z - max z)) in units, sum e
    float m, s, cross, share;
};

struct RingLate {  // a row whose entries' columns are written after all others
    int row, kind;  // kind 0: nothing to write, 1: every column is named once, 2: some more than once
    float m, scale, taken, top, sum;
};

template <int WORKERS>
struct RingShared {
    MaxSum part[kMostSlots][WORKERS / 32];
    RingRow row[kMostSlots];
    int vectors[kMostSlots];
    alignas(16) RingBlock block[2][kDistillMostCtas];
    float v[3][kListed];  // the entries of this row and the next two; at last what becomes of their columns
    int col[3][kListed];
    alignas(8) unsigned long long full[kMostSlots];  // a slot's copies have arrived
    alignas(8) unsigned long long told[2];           // the blocks of a row have
    int dead;                                        // something did not within the limit: from there on the loss and gradient of every row are NaN
    int joined;                                      // rows whose sums the manager has taken
    RingLate late[kMostRows];
};

// Barriers of the CTA by number, for `threads` threads: arriving does not wait.
__device__ __forceinline__ void barrier_arrive(int number, int threads) { asm volatile("barrier.cta.arrive %0, %1;" ::"r"(number), "r"(threads) : "memory"); }
__device__ __forceinline__ void barrier_sync(int number, int threads) { asm volatile("barrier.cta.sync %0, %1;" ::"r"(number), "r"(threads) : "memory"); }

// 16 bytes to the same place in the shared memory of CTA `rank` of the cluster, counted by its barrier
__device__ __forceinline__ void tell(unsigned to, const RingBlock& b, unsigned bar, int rank)
{
    asm volatile(
        "{\n\t.reg .b32 ra, rb;\n\t"
        "mapa.shared::cluster.u32 ra, %0, %6;\n\t"
        "mapa.shared::cluster.u32 rb, %1, %6;\n\t"
        "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [ra], {%2, %3, %4, %5}, [rb];\n\t}" ::"r"(to),
        "r"(bar), "r"(__float_as_uint(b.m)), "r"(__float_as_uint(b.s)), "r"(__float_as_uint(b.cross)), "r"(__float_as_uint(b.share)), "r"(rank)
        : "memory");
}

// Grid: clusters of 2^log_parts CTAs, each with `rows` rows in turn.
template <class T, int WORKERS, bool GRADIENT>
__global__ void __launch_bounds__(WORKERS + 32, WORKERS == 128 ? 6 : WORKERS == 256 ? 3 : 1) distill_ring_kernel(DistillParams p)
{
    constexpr int N = Part<T>::N, W = WORKERS / 32, UNROLL = 4, ALL = WORKERS + 32;
    constexpr int kSums = 1, kRow = 1 + kMostSlots, kWritten = 1 + 2 * kMostSlots;  // barriers, one a slot each
    __shared__ RingShared<WORKERS> sh;
    extern __shared__ __align__(128) unsigned char ring_smem[];
    unsigned* named = reinterpret_cast<unsigned*>(ring_smem);  // GRADIENT: a bit for each column of the part
    unsigned char* ring = ring_smem + p.ring_offset;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int first_row = (int)(blockIdx.x >> p.log_parts) * p.rows;
    const int rows = min(p.rows, p.T - first_row), parts = 1 << p.log_parts;
    const float c = p.inv_t * CUDART_L2E_F;
    volatile int* const dead = &sh.dead;

    if (tid == 0) {
        for (int k = 0; k < p.slots; ++k) mbar_init(smem_u32(&sh.full[k]), 1);
        for (int k = 0; k < 2; ++k) mbar_init(smem_u32(&sh.told[k]), 1);
        sh.dead = 0;
        sh.joined = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if constexpr (GRADIENT) {
        for (int i = tid; i * 4 < p.ring_offset; i += ALL) named[i] = 0;
    }
    wait_for_previous_grid();
    if (parts > 1) cooperative_groups::this_cluster().sync();  // the others' barriers are there
    else __syncthreads();

    if (warp < W) {  // ---- workers
        int slot = 0;
        unsigned phase = 0;
        for (int i = 0; i < rows; ++i) {
            bool arrived = *dead == 0;
            if (arrived) {
                arrived = mbar_wait_bounded(smem_u32(&sh.full[slot]), phase, kWalkFactor * p.wait_limit);
                if (!arrived) *dead = 1;
            }
            if (!arrived) {  // without copies to wait for, no further ahead of the manager than they would let this warp be
                volatile int* const joined = &sh.joined;
                for (unsigned spin = 0; spin < kToldLimit && *joined + p.slots <= i; ++spin) {}
            }
            __syncwarp();
            const uint4* const from = reinterpret_cast<const uint4*>(ring + slot * p.slot_bytes);
            const int vectors = arrived ? sh.vectors[slot] : 0;
            constexpr unsigned none = Words<T>::kMinusInf;
            unsigned top_words = none;
            for (int k = tid; k < vectors; k += UNROLL * WORKERS) {
                uint4 v[UNROLL];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) v[u] = k + u * WORKERS < vectors ? from[k + u * WORKERS] : make_uint4(none, none, none, none);
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) top_words = max_words<T>(top_words, v[u]);
            }
            const Exponent y(warp_max(fmaxf(Words<T>::largest(top_words), kLowest)), c);
            Pair sum = pair_of(0.0f, 0.0f);
            const auto add = [&](auto far) {
                const auto take = [&](const uint4& v) {
                    Words<T>::each(v, [&](Pair w) { sum = add2(sum, exp2_approx(y.template of<decltype(far)::value>(w))); });
                };
                int k = tid;
                for (; k + (UNROLL - 1) * WORKERS < vectors; k += UNROLL * WORKERS) {
                    uint4 v[UNROLL];
#pragma unroll
                    for (int u = 0; u < UNROLL; ++u) v[u] = from[k + u * WORKERS];
#pragma unroll
                    for (int u = 0; u < UNROLL; ++u) take(v[u]);
                }
                for (; k < vectors; k += WORKERS) take(from[k]);
            };
            if (y.far) add(std::true_type());
            else add(std::false_type());
            const float s = warp_sum(arrived ? halves(sum).x + halves(sum).y : CUDART_NAN_F);
            if (lane == 0) sh.part[slot][warp] = {y.m, s};
            barrier_arrive(kSums + slot, ALL);
            if constexpr (GRADIENT) {
                barrier_sync(kRow + slot, ALL);
                const RingRow row = sh.row[slot];
                T* const to = static_cast<T*>(row.to);
                if (row.zero || !arrived) {
                    const unsigned word = row.zero ? 0u : Words<T>::kNaN;
                    for (int k = tid; k < row.vectors; k += WORKERS) store_vector(to + (long long)k * N, make_uint4(word, word, word, word), row.aligned);
                } else {
                    const Exponent z(row.m, c);
                    const auto write = [&](auto far) {
                        const Pair scale = pair_of(row.scale, row.scale);
                        const auto value = [&](Pair v) { return mul2(scale, exp2_approx(z.template of<decltype(far)::value>(v))); };
#pragma unroll 4
                        for (int k = tid; k < vectors; k += WORKERS) store_vector(to + (long long)k * N, Words<T>::map(from[k], value), row.aligned);
                    };
                    if (z.far) write(std::true_type());
                    else write(std::false_type());
                }
                barrier_arrive(kWritten + slot, ALL);
            }
            if (++slot == p.slots) slot = 0, phase ^= 1;
        }
    } else {  // ---- the manager
        const int rank = (int)blockIdx.x & (parts - 1);
        const T* const all_x = static_cast<const T*>(p.x);
        int issued = 0;
        const auto issue = [&](int i, int slot) {  // the copies of row first_row + i
            ++issued;
            const Place at(p, first_row + i);
            const T* x = all_x + (long long)at.row * p.ldx;
            const Part<T> part(x, at.c0, at.c1);
            if (lane == 0) {
                const unsigned bar = smem_u32(&sh.full[slot]), to = smem_u32(ring + slot * p.slot_bytes), bytes = (unsigned)part.vectors * 16u;
                sh.vectors[slot] = part.vectors;
                mbar_expect_tx(bar, bytes);
                constexpr unsigned kPiece = 16384;
                for (unsigned from = 0; from < bytes; from += kPiece)
                    bulk_copy_g2s(to + from, reinterpret_cast<const char*>(x + part.first) + from, min(kPiece, bytes - from), bar);
            }
        };
        for (int i = 0; i < min(p.slots, rows); ++i) issue(i, i);
        // Row offsets are asked for four rows ahead, entries two and the part's single elements (a lane each) and the weight one row ahead; a
        // row's shares are made while the workers write the row before it.
        const auto offset = [&](int i) { return __ldg(p.row_ptr + first_row + min(i, rows)); };
        int offsets[5] = {offset(0), offset(1), offset(2), offset(3), 0};  // of row i and the next ones
        const auto fetch_entries = [&](int i, int from, int to) {
            const Teacher t = teacher_of(p, from, to);
            const int buffer = i % 3;
            if (i < rows && t.count <= kListed) {
                for (int j = lane; j < t.count; j += 32) {
                    async_copy_vec<1>(smem_u32(&sh.v[buffer][j]), t.v + j);
                    async_copy_vec<1>(smem_u32(&sh.col[buffer][j]), t.cols + j);
                }
            }
            async_commit();
        };
        const auto edge_column = [&](const Part<T>& part, const Place& at) {
            const int head = part.first - at.c0, behind = part.first + part.vectors * N + lane - head;
            return lane < head ? at.c0 + lane : behind < at.c1 ? behind : -1;
        };
        const auto fetch_edge = [&](int i) {
            const Place at(p, first_row + i);
            const T* x = all_x + (long long)at.row * p.ldx;
            const int col = edge_column(Part<T>(x, at.c0, at.c1), at);
            return col >= 0 ? to_f32(x[col]) : -CUDART_INF_F;
        };
        const auto value_of = [&](const Teacher& t, int i, int j) { return t.count <= kListed ? sh.v[i % 3][j] : __ldg(t.v + j); };
        const float unit = cross_unit(p);
        const auto over_of = [&](const Teacher& t, float v) { return p.log_probs ? v : (v - t.top) * p.inv_t; };
        const auto teach = [&](int i, int from, int to) {  // row i's shares: exp(over_of) / sum; top is -infinity where none weighs anything
            Teacher t = teacher_of(p, from, to);
            t.top = -CUDART_INF_F;
            t.sum = 0.0f;
            async_wait<1>();  // all but the latest fetch
            __syncwarp();
            if (p.log_probs) {
                if (t.count > 0) t.top = 0.0f;
            } else {
                bool broken = false;
#pragma unroll 4
                for (int j = lane; j < t.count; j += 32) {
                    const float v = value_of(t, i, j);
                    t.top = fmaxf(t.top, v);
                    broken |= v != v;
                }
                t.top = __any_sync(kAllLanes, broken) ? CUDART_NAN_F : warp_max(t.top);
            }
            if (t.top != -CUDART_INF_F) {
#pragma unroll 4
                for (int j = lane; j < t.count; j += 32) t.sum += expf(over_of(t, value_of(t, i, j)));
                t.sum = warp_sum(t.sum);
            }
            return t;
        };
        const auto weight_of = [&](int i) { return GRADIENT ? __ldg(p.weight + (first_row + i) * p.weight_stride) : 0.0f; };
        fetch_entries(0, offsets[0], offsets[1]);
        fetch_entries(1, offsets[1], offsets[2]);
        float next_edge = fetch_edge(0), next_weight = weight_of(0);
        Teacher next = teach(0, offsets[0], offsets[1]);
        int slot = 0, late = 0;
        unsigned phase = 0;
        for (int i = 0; i < rows; ++i) {
            const Place at(p, first_row + i);
            const T* x = all_x + (long long)at.row * p.ldx;
            const Part<T> part(x, at.c0, at.c1);
            const T* const here = reinterpret_cast<const T*>(ring + slot * p.slot_bytes);
            const auto element = [&](int col) {  // of this part
                const int k = col - part.first;
                return to_f32(k >= 0 && k < part.vectors * N ? here[k] : x[col]);
            };
            const Teacher t = next;
            const bool listed = t.count <= kListed, counts = t.top != -CUDART_INF_F;
            const auto column = [&](int j) { return listed ? min(max(sh.col[i % 3][j], 0), p.V - 1) : t.column(p, j); };
            const float edge = next_edge, weight = next_weight;
            offsets[4] = offset(i + 4);

            // While the workers sum.  The entries of the part's columns, relative to the largest of the student's logits there, and the single
            // elements of the lanes.
            bool arrived = *dead == 0;
            if (arrived) {
                arrived = mbar_wait_bounded(smem_u32(&sh.full[slot]), phase, p.wait_limit);
                if (!arrived) *dead = 1;
            }
            arrived = __all_sync(kAllLanes, arrived);
            float cross = 0.0f, share = 0.0f, top = kLowest;
            if (counts) {
                for (int j = lane; j < t.count; j += 32) {
                    const int col = column(j);
                    if (col >= at.c0 && col < at.c1) top = fmaxf(top, element(col));
                }
                top = warp_max(top);
                const Exponent y(top, c);
                for (int j = lane; j < t.count; j += 32) {
                    const int col = column(j);
                    if (col >= at.c0 && col < at.c1) {
                        const float over = over_of(t, value_of(t, i, j)), e = expf(over);
                        share += e;
                        if (e != 0.0f) cross += e * ((over - y.below(element(col), p.inv_t)) * unit);
                    }
                }
                cross = warp_sum(cross);
                share = warp_sum(share);
            }
            MaxSum edges = {fmaxf(warp_max(edge), kLowest), 0.0f};
            edges.s = warp_sum(exp2_approx(Exponent(edges.m, c).of(edge)));

            // the part's maximum and sum
            barrier_sync(kSums + slot, ALL);
            if (lane == 0) *const_cast<volatile int*>(&sh.joined) = i + 1;
            constexpr int kJoined = W < 16 ? 16 : 32;
            const int whose = lane % kJoined;
            MaxSum mine = join_lanes<kJoined>(whose < W ? sh.part[slot][whose] : whose == W ? edges : MaxSum{kLowest, 0.0f}, c);
            if (!arrived) mine.s = CUDART_NAN_F;
            if (share != 0.0f) cross -= Exponent(mine.m, c).max_below(top, p.inv_t) * unit * share;
            if constexpr (!GRADIENT) {
                if (arrived && i + p.slots < rows) {  // everybody has read the slot
                    if (lane == 0) fence_proxy_async_smem();
                    issue(i + p.slots, slot);
                }
            }

            // the row's: every part tells every other
            RingBlock block = {mine.m, mine.s, cross, share};
            MaxSum all = mine;
            if (parts > 1) {
                const unsigned bar = smem_u32(&sh.told[i & 1]);
                if (lane == 0) mbar_expect_tx(bar, (unsigned)parts * sizeof(RingBlock));
                if (lane < parts) tell(smem_u32(&sh.block[i & 1][rank]), block, bar, lane);
                bool told = *dead == 0 && mbar_wait_bounded(bar, (unsigned)(i >> 1) & 1u, kToldLimit);
                told = __all_sync(kAllLanes, told);
                if (!told) *dead = 1;
                block = lane % 8 < parts ? sh.block[i & 1][lane % 8] : RingBlock{kLowest, 0.0f, 0.0f, 0.0f};
                all = join_lanes<8>({block.m, block.s}, c);
                if (!told) all.s = CUDART_NAN_F;
            }
            const Exponent y(all.m, c);
            const float mass = !counts ? 0.0f : p.log_probs || t.sum != t.sum ? t.sum : 1.0f;
            const bool zero = mass == 0.0f;
            const float scale = weight * p.temperature * mass / all.s;
            if constexpr (GRADIENT) {
                T* const to = static_cast<T*>(p.dx) + (long long)at.row * p.ldd + part.first;
                if (lane == 0) sh.row[slot] = {all.m, scale, zero, (reinterpret_cast<uintptr_t>(to) & 15u) == 0, part.vectors, to};
                barrier_arrive(kRow + slot, ALL);
            }

            // while the workers write
            fetch_entries(i + 2, offsets[2], offsets[3]);
            if (i + 1 < rows) {
                next_edge = fetch_edge(i + 1);
                next_weight = weight_of(i + 1);
            }
            if (rank == 0) {
                float crosses = 0.0f;
                if (lane < parts) crosses = block.cross - (block.share != 0.0f ? y.max_below(block.m, p.inv_t) * unit * block.share : 0.0f);
                crosses = warp_sum(crosses);
                if (lane == 0) {
                    const float lse = logf(all.s), tt = p.temperature * p.temperature;
                    p.loss[at.row] = zero ? 0.0f : tt * divergence(p, crosses, t.sum, mass, lse);
                    if (p.stats != nullptr)
                        p.stats[at.row] = counts ? make_float4(all.m, all.s, t.top, t.sum) : make_float4(0.0f, 1.0f, -CUDART_INF_F, 1.0f);
                }
            }
            if constexpr (GRADIENT) {
                T* const out = static_cast<T*>(p.dx) + (long long)at.row * p.ldd;
                const int edge_col = edge_column(part, at);
                if (edge_col >= 0) out[edge_col] = from_f32<T>(zero ? 0.0f : scale * exp2_approx(y.of(edge)));
                const auto share_of = [&](int j) {
                    const float e = expf(over_of(t, value_of(t, i, j)));
                    return p.log_probs ? e : e / t.sum;
                };
                const auto gradient = [&](int col, float taken) {
                    return scale * exp2_approx(y.of(element(col))) - weight * p.temperature * taken;
                };
                const auto inside = [&](int col) { return !zero && col >= at.c0 && col < at.c1; };
                // whether entry j's column is marked before
                const auto marked = [&](int j) {
                    const int col = column(j), k = col - at.c0;
                    return inside(col) && ((atomicOr(&named[k >> 5], 1u << (k & 31)) >> (k & 31)) & 1u) != 0;
                };
                const auto unmark = [&] {
                    __syncwarp();
                    for (int j = lane; j < t.count; j += 32)
                        if (inside(column(j))) named[(column(j) - at.c0) >> 5] = 0;
                };
                bool repeats = false;
                if (!zero) {
                    for (int j = lane; j < t.count; j += 32) repeats |= marked(j);
                    repeats = __any_sync(kAllLanes, repeats);
                    unmark();
                }
                if (listed && !repeats) {  // what becomes of a list's columns is known before the workers are done
                    for (int j = lane; j < t.count; j += 32)
                        if (inside(column(j))) sh.v[i % 3][j] = gradient(column(j), share_of(j));
                } else if (listed) {  // columns that are named again, one at a time, with all their p, whichever of their entries marks them first
                    __syncwarp();
                    unsigned again = 0, done = 0;
                    for (int j = lane; j < t.count; j += 32) again |= (unsigned)marked(j) << (j / 32);
                    unmark();
                    for (unsigned left; (left = __ballot_sync(kAllLanes, again != 0)) != 0; again &= ~done) {
                        const int whose = __ffs(left) - 1, col = column(__shfl_sync(kAllLanes, __ffs(again) - 1, whose) * 32 + whose);
                        float taken = 0.0f;
                        for (int j = lane; j < t.count; j += 32)
                            if (column(j) == col) taken += share_of(j);
                        const float g = gradient(col, warp_sum(taken));
                        for (int j = lane; j < t.count; j += 32)
                            if (column(j) == col) sh.v[i % 3][j] = g, done |= 1u << (j / 32);
                    }
                    for (int j = lane; j < t.count; j += 32)
                        if (inside(column(j)) && !((done >> (j / 32)) & 1u)) sh.v[i % 3][j] = gradient(column(j), share_of(j));
                }
                if (i + 1 < rows) next = teach(i + 1, offsets[1], offsets[2]);
                barrier_sync(kWritten + slot, ALL);  // what the workers wrote comes before what is written here
                if (!listed) {
                    if (repeats || t.count > kLongWalk) {
                        if (lane == 0) sh.late[late] = {at.row, zero ? 0 : repeats ? 2 : 1, y.m, scale, weight * p.temperature, t.top, t.sum};
                        ++late;
                    } else {
                        for (int j = lane; j < t.count; j += 32)
                            if (inside(column(j))) out[column(j)] = from_f32<T>(gradient(column(j), share_of(j)));
                        __syncwarp();
                    }
                }
                if (arrived && i + p.slots < rows) {  // everybody has read the slot
                    if (lane == 0) fence_proxy_async_smem();
                    issue(i + p.slots, slot);
                }
                if (listed) {
                    for (int j = lane; j < t.count; j += 32)
                        if (inside(column(j))) out[column(j)] = from_f32<T>(sh.v[i % 3][j]);
                }
                __syncwarp();  // the row's entries have been read
            } else if (i + 1 < rows) {
                next = teach(i + 1, offsets[1], offsets[2]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) offsets[k] = offsets[k + 1];
            if (++slot == p.slots) slot = 0, phase ^= 1;
        }
        async_wait<0>();
        if constexpr (GRADIENT) {
            __syncwarp();
            for (int k = 0; k < late; ++k) {  // nobody waits for these
                const RingLate l = sh.late[k];
                const Place at(p, l.row);
                Teacher t = teacher_of(p, __ldg(p.row_ptr + l.row), __ldg(p.row_ptr + l.row + 1));
                t.top = l.top;
                t.sum = p.log_probs ? 1.0f : l.sum;
                const T* const x = all_x + (long long)l.row * p.ldx;
                T* const out = static_cast<T*>(p.dx) + (long long)l.row * p.ldd;
                if (l.kind == 2) {  // the bits are as many as a 32nd of the columns: 32 walks over the entries
                    write_named_columns<T, 4>({reinterpret_cast<float*>(named), p.ring_offset / 4, 0, 1, at.c0, at.c1, p.V, t, p.log_probs, p.inv_t, c, l.m,
                                               l.scale, l.taken, x, out});
                } else if (l.kind == 1) {
                    const Exponent y(l.m, c);
                    for (int j = lane; j < t.count; j += 32) {
                        const int col = t.column(p, j);
                        if (col >= at.c0 && col < at.c1) out[col] = from_f32<T>(l.scale * exp2_approx(y.of(to_f32(x[col]))) - l.taken * t.share(p, __ldg(t.v + j)));
                    }
                }
            }
        }
        if (*dead != 0 && lane == 0) {  // no copy may arrive after the CTA has gone
            for (int i = max(issued - p.slots, 0); i < issued; ++i) mbar_wait_bounded(smem_u32(&sh.full[i % p.slots]), (unsigned)(i / p.slots) & 1u);
        }
    }
    if (parts > 1) cooperative_groups::this_cluster().sync();  // nobody leaves while another may still tell it something
}

// Rows longer than a cluster holds: the same in two sweeps over the part, the second from L2 where it has stayed there.
constexpr int kLongThreads = 512;
constexpr int kLongUnroll = 4;

template <class T, bool GRADIENT>
__global__ void __launch_bounds__(kLongThreads, 2) distill_long_kernel(DistillParams p)
{
    constexpr int N = Part<T>::N, THREADS = kLongThreads;
    constexpr int kSpan = 512;
    __shared__ Room<THREADS> room;
    __shared__ union {
        unsigned named[THREADS / 32 * kSpan];
        float sums[THREADS / 32 * kSpan];
    } sh;
    wait_for_previous_grid();
    const Place at(p);
    const T* x = static_cast<const T*>(p.x) + (long long)at.row * p.ldx;
    const Part<T> part(x, at.c0, at.c1);
    Teacher t = teacher_of(p, __ldg(p.row_ptr + at.row), __ldg(p.row_ptr + at.row + 1));
    if (t.count == 0) {
        leave_out<T, THREADS>(p, at, true, GRADIENT);
        return;
    }
    const Entries<T, THREADS> entries(p, t, x);
    const float c = p.inv_t * CUDART_L2E_F;
    const float edge = part.edge >= 0 ? to_f32(x[part.edge]) : -CUDART_INF_F;
    const auto load = [&](int k, uint4 (&v)[kLongUnroll]) {
        constexpr unsigned none = Words<T>::kMinusInf;
#pragma unroll
        for (int u = 0; u < kLongUnroll; ++u)
            v[u] = k + u * THREADS < part.vectors ? __ldg(reinterpret_cast<const uint4*>(x + part.first) + k + u * THREADS) : make_uint4(none, none, none, none);
    };

    MaxSum mine = {kLowest, 0.0f};
    for (int k = threadIdx.x; k < part.vectors; k += kLongUnroll * THREADS) {
        uint4 v[kLongUnroll];
        load(k, v);
        unsigned top_words = v[0].x;
#pragma unroll
        for (int u = 0; u < kLongUnroll; ++u) top_words = max_words<T>(top_words, v[u]);
        const Exponent y(fmaxf(mine.m, Words<T>::largest(top_words)), c);
        if (y.m > mine.m) mine = {y.m, mine.s * exp2_approx(y.of_max(mine.m))};
        Pair sum = pair_of(0.0f, 0.0f);
        const auto add = [&](auto far) {
#pragma unroll
            for (int u = 0; u < kLongUnroll; ++u)
                Words<T>::each(v[u], [&](Pair w) { sum = add2(sum, exp2_approx(y.template of<decltype(far)::value>(w))); });
        };
        if (y.far) add(std::true_type());
        else add(std::false_type());
        mine.s += halves(sum).x + halves(sum).y;
    }
    if (part.edge >= 0) {
        const Exponent y(fmaxf(mine.m, edge), c);
        mine = {y.m, mine.s * exp2_approx(y.of_max(mine.m)) + exp2_approx(y.of(edge))};
    }
    if (!p.log_probs) leave_top<T, THREADS>(entries, room);
    const MaxSum all = join_row<THREADS>(join_lanes<32>(mine, c), c, room, p.log_parts);
    if (!p.log_probs) {
        t.top = joined_top<THREADS>(room);
        if (t.top == -CUDART_INF_F) {
            leave_out<T, THREADS>(p, at, true, GRADIENT);
            leave_row(p.log_parts);
            return;
        }
    }
    const Exponent y(all.m, c);
    const float mass = finish_loss<T, THREADS>(p, at, entries, t, y, all.s, room);
    if constexpr (GRADIENT) {
        T* out = static_cast<T*>(p.dx) + (long long)at.row * p.ldd;
        if (mass == 0.0f) {
            zero_part<T, THREADS>(out, at.c0, at.c1);
        } else {
            const float weight = __ldg(p.weight + at.row * p.weight_stride);
            const float scale = weight * p.temperature * mass / all.s;
            T* to = out + part.first;
            const bool aligned = (reinterpret_cast<uintptr_t>(to) & 15u) == 0;
            const auto value = [&](Pair v) {
                const float2 w = halves(v);
                return mul2(pair_of(scale, scale), exp2_approx(pair_of(y.of(w.x), y.of(w.y))));
            };
            for (int k = threadIdx.x; k < part.vectors; k += kLongUnroll * THREADS) {
                uint4 v[kLongUnroll];
                load(k, v);
#pragma unroll
                for (int u = 0; u < kLongUnroll; ++u)
                    if (k + u * THREADS < part.vectors) store_vector(to + (long long)(k + u * THREADS) * N, Words<T>::map(v[u], value), aligned);
            }
            if (part.edge >= 0) out[part.edge] = from_f32<T>(scale * exp2_approx(y.of(edge)));
            // ascending columns name none twice; of others the part's are marked, a bit each, as many at once as there is room for
            bool repeats = false;
            for (int i = threadIdx.x; i + 1 < t.count; i += THREADS) repeats |= t.column(p, i) >= t.column(p, i + 1);
            if (__syncthreads_or(repeats)) {
                constexpr int kMarked = THREADS * kSpan;
                repeats = false;
                for (long long base = at.c0; base < at.c1; base += kMarked) {
                    for (int i = threadIdx.x; i < kMarked / 32; i += THREADS) sh.named[i] = 0;
                    __syncthreads();
                    for (int i = threadIdx.x; i < t.count; i += THREADS) {
                        const long long k = t.column(p, i) - base;
                        if (k >= 0 && k < min((long long)kMarked, at.c1 - base)) repeats |= (atomicOr(&sh.named[k >> 5], 1u << (k & 31)) >> (k & 31)) & 1u;
                    }
                    repeats = __syncthreads_or(repeats);
                    if (repeats) break;
                }
            }
            write_entries<T, THREADS>(p, entries, t, y, scale, weight, out, at.c0, at.c1, repeats, sh.sums, kSpan);
        }
    }
    leave_row(p.log_parts);
}

}  // namespace csrspmm_b200

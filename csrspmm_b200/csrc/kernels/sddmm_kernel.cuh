// The gradient of C = alpha * A * B for A's stored values: out[e] = alpha * <G[row(e), :], B[col(e), :]> for every stored entry e
// (a dense product sampled at the matrix's pattern).  The reference has no gradients.
//
// A CTA takes a run of consecutive entries, so that rows of any length are split evenly and a row of G is read
// by the lanes that need it next to one another.  It finds the rows of its run once: the first and the last by a search
// that 32 lanes make together, those between from their offsets.  L lanes then own an entry at a time and hold NV vectors of
// the row of G in registers for as long as the row stays the same; the rows of B are asked for U entries ahead.
// Every entry is one sum in a fixed order: no atomics.
#pragma once

#include <climits>

#include "common.cuh"
#include "score_types.cuh"

namespace csrspmm_b200 {

constexpr int kSddmmThreads = 256;
constexpr int kSddmmMostEntries = 1024;  // of a CTA's run

struct SddmmParams {
    int M, Kd, nvec;  // columns in vectors of VW
    int nnz;
    const int* row_ptr;
    const int* col_idx;
    const float* G;
    long long ldg;
    const float* B;
    long long ldb;
    float alpha;
    int run;  // entries of a CTA, a multiple of its groups of lanes
    float* out;
};

// Steps of 32 that cover `rows` rows, of which there may be 2^31 - 1.
__host__ __device__ constexpr int search_step(int rows) { return (rows - 1) / 32 + 1; }
static_assert(search_step(2) == 1 && search_step(33) == 2 && search_step(INT_MAX) == 1 << 26, "whole steps, without passing 32 bits");

// The last row r of [0, M) with row_ptr[r] <= e (0 where there is none), by all lanes of a warp.
__device__ __forceinline__ int row_of_entry(const int* row_ptr, int M, int e, int lane)
{
    int lo = 0, hi = M;  // the answer is in [lo, hi)
    while (hi - lo > 1) {
        const int step = search_step(hi - lo);
        const long long at = lo + (long long)lane * step;
        const bool at_or_before = at < hi && (lane == 0 || __ldg(row_ptr + at) <= e);
        const int last = 31 - __clz(__ballot_sync(kAllLanes, at_or_before));
        const int from = lo + last * step;
        hi = hi - from > step ? from + step : hi;
        lo = from;
    }
    return lo;
}

template <int VW>
__device__ __forceinline__ float dot(const Vec<VW>& a, const Vec<VW>& b, float sum)
{
    if constexpr (VW == 4) {
        sum = __fmaf_rn(a.v.x, b.v.x, sum);
        sum = __fmaf_rn(a.v.y, b.v.y, sum);
        sum = __fmaf_rn(a.v.z, b.v.z, sum);
        return __fmaf_rn(a.v.w, b.v.w, sum);
    } else if constexpr (VW == 2) {
        sum = __fmaf_rn(a.v.x, b.v.x, sum);
        return __fmaf_rn(a.v.y, b.v.y, sum);
    } else {
        return __fmaf_rn(a.v, b.v, sum);
    }
}

// A vector of a row of B that is too wide to be met again in L1: kept out of it, where G's row serves several entries (a training step of
// 4096 rows of 8 entries, 2048 columns: 213 -> 205 us).  Narrow rows are left in: on a graph that is worth more than the room (262 144 rows of 16, 128 columns: 220 against 306 us).
__device__ __forceinline__ void load_past_l1(Vec<4>& r, const float* p)
{
    asm("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(r.v.x), "=f"(r.v.y), "=f"(r.v.z), "=f"(r.v.w) : "l"(p));
}
__device__ __forceinline__ void load_past_l1(Vec<2>& r, const float* p)
{
    asm("ld.global.nc.L1::no_allocate.v2.f32 {%0, %1}, [%2];" : "=f"(r.v.x), "=f"(r.v.y) : "l"(p));
}
__device__ __forceinline__ void load_past_l1(Vec<1>& r, const float* p) { asm("ld.global.nc.L1::no_allocate.f32 %0, [%1];" : "=f"(r.v) : "l"(p)); }

// LOOP: rows wider than L * NV vectors, in steps of that many
template <int L, int NV, int VW, bool LOOP>
__global__ void __launch_bounds__(kSddmmThreads) sddmm_kernel(SddmmParams p)
{
    constexpr int kGroups = kSddmmThreads / L;
    constexpr int U = LOOP ? 1 : NV == 4 ? 2 : NV == 2 ? 4 : 8;  // rows of B asked for at once: eight vectors
    __shared__ int row_of[kSddmmMostEntries];
    __shared__ int warp_last[kSddmmThreads / 32];
    __shared__ int bounds[2];
    wait_for_previous_grid();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long begin = (long long)blockIdx.x * p.run;
    const int n = (int)min((long long)p.run, (long long)p.nnz - begin);
    if (warp < 2) {
        const int r = row_of_entry(p.row_ptr, p.M, (int)(begin + (warp == 0 ? 0 : n - 1)), lane);
        if (lane == 0) bounds[warp] = r;
    }
    for (int i = tid; i < kSddmmMostEntries; i += kSddmmThreads) row_of[i] = 0;
    __syncthreads();
    const int r0 = bounds[0], r1 = bounds[1];
    for (long long r = r0 + 1LL + tid; r <= r1; r += kSddmmThreads) {  // where the rows after the first begin; of empty ones the last counts
        const long long at = (long long)__ldg(p.row_ptr + r) - begin;
        if (at >= 0 && at < n) atomicMax(&row_of[at], (int)(r - r0));
    }
    __syncthreads();
    {  // running maximum over the run, kEach entries a thread
        constexpr int kEach = kSddmmMostEntries / kSddmmThreads;
        int mine[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) mine[i] = i > 0 ? max(mine[i - 1], row_of[kEach * tid + i]) : row_of[kEach * tid];
        int upto = mine[kEach - 1];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(kAllLanes, upto, d);
            if (lane >= d) upto = max(upto, v);
        }
        if (lane == 31) warp_last[warp] = upto;
        int before = __shfl_up_sync(kAllLanes, upto, 1);
        if (lane == 0) before = 0;
        __syncthreads();
        for (int w = 0; w < warp; ++w) before = max(before, warp_last[w]);
#pragma unroll
        for (int i = 0; i < kEach; ++i) row_of[kEach * tid + i] = r0 + max(before, mine[i]);
    }
    __syncthreads();

    const int group = tid / L, gl = tid % L;
    const int per_group = p.run / kGroups;
    const int first = group * per_group, end = min(first + per_group, n);
    // lanes of a warp shuffle together: all groups make the same number of steps
    Vec<VW> g[NV];
    int held = -1;
    for (int s = 0; s < per_group; s += U) {
        if constexpr (!LOOP) {
            Vec<VW> b[U][NV];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = first + s + u;
                if (s + u < per_group && i < end) {
                    const int col = min(max(__ldg(p.col_idx + begin + i), 0), p.Kd - 1);
                    const float* from = p.B + (long long)col * p.ldb;
#pragma unroll
                    for (int v = 0; v < NV; ++v) {
                        if (gl + v * L < p.nvec) b[u][v].load_nc(from + (gl + v * L) * VW);
                        else b[u][v].zero();
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = first + s + u;
                const bool there = s + u < per_group && i < end;
                float sum = 0.0f;
                if (there) {
                    const int row = row_of[i];
                    if (row != held) {
                        held = row;
                        const float* from = p.G + (long long)row * p.ldg;
#pragma unroll
                        for (int v = 0; v < NV; ++v) {
                            if (gl + v * L < p.nvec) g[v].load_nc(from + (gl + v * L) * VW);
                            else g[v].zero();
                        }
                    }
#pragma unroll
                    for (int v = 0; v < NV; ++v) sum = dot(g[v], b[u][v], sum);
                }
#pragma unroll
                for (int d = L / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(kAllLanes, sum, d);
                if (there && gl == 0) p.out[begin + i] = p.alpha * sum;
            }
        } else {
            const int i = first + s;
            float sum = 0.0f;
            if (i < end) {
                const int col = min(max(__ldg(p.col_idx + begin + i), 0), p.Kd - 1);
                const float* fb = p.B + (long long)col * p.ldb;
                const float* fg = p.G + (long long)row_of[i] * p.ldg;
                for (int c = gl; c < p.nvec; c += L * NV) {
                    Vec<VW> b[NV];
#pragma unroll
                    for (int v = 0; v < NV; ++v) {
                        if (c + v * L < p.nvec) {
                            load_past_l1(b[v], fb + (c + v * L) * VW);
                            g[v].load_nc(fg + (c + v * L) * VW);
                        } else {
                            b[v].zero();
                            g[v].zero();
                        }
                    }
#pragma unroll
                    for (int v = 0; v < NV; ++v) sum = dot(g[v], b[v], sum);
                }
            }
#pragma unroll
            for (int d = L / 2; d > 0; d >>= 1) sum += __shfl_xor_sync(kAllLanes, sum, d);
            if (i < end && gl == 0) p.out[begin + i] = p.alpha * sum;
        }
    }
}

// ---- the gradient for B of a small product -----------------------------------------------------------------
//
// C = alpha * A^T * G without a transpose: a warp owns a row of C (a column of A) and up to 32 * kTransposedVectors vectors of its columns, looks
// through all of A's columns and adds up the entries that are its own, in stored order.  That reads nnz columns Kd times, and takes one
// launch where transposition and product take seven: what a small training step costs is those launches.

constexpr int kTransposedThreads = 256;
constexpr int kTransposedVectors = 4;

struct TransposedParams {
    int M, Kd, nvec, nnz;
    const int* row_ptr;
    const int* col_idx;
    const float* values;
    const float* G;
    long long ldg;
    float alpha;
    float* C;
    long long ldc;
};

template <int VW>
__global__ void __launch_bounds__(kTransposedThreads) spmm_transposed_kernel(TransposedParams p)
{
    constexpr int NV = kTransposedVectors, U = 4;
    wait_for_previous_grid();
    const int lane = threadIdx.x & 31;
    const long long own = (long long)blockIdx.x * (kTransposedThreads / 32) + (threadIdx.x >> 5);  // row of C and part of its columns
    const int parts = (p.nvec + 32 * NV - 1) / (32 * NV);
    const int row = (int)(own / parts), v0 = (int)(own % parts) * 32 * NV + lane;
    if (row >= p.Kd) return;
    Vec<VW> sum[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) sum[k].zero();
    for (int base = 0; base < p.nnz; base += 32 * U) {
        int col[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long e = (long long)base + u * 32 + lane;
            col[u] = e < p.nnz ? min(max(__ldg(p.col_idx + e), 0), p.Kd - 1) : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            unsigned mine = __ballot_sync(kAllLanes, col[u] == row);
            for (; mine != 0; mine &= mine - 1) {
                const int e = base + u * 32 + __ffs(mine) - 1;
                const float* from = p.G + (long long)row_of_entry(p.row_ptr, p.M, e, lane) * p.ldg;
                const float value = __ldg(p.values + e);
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    if (v0 + k * 32 < p.nvec) {
                        Vec<VW> g;
                        g.load_nc(from + (long long)(v0 + k * 32) * VW);
                        sum[k].fma(value, g);
                    }
                }
            }
        }
        if (base > INT_MAX - 32 * U) break;
    }
    float* const to = p.C + (long long)row * p.ldc;
#pragma unroll
    for (int k = 0; k < NV; ++k)
        if (v0 + k * 32 < p.nvec) sum[k].epilogue0(p.alpha).store(to + (long long)(v0 + k * 32) * VW);
}

}  // namespace csrspmm_b200

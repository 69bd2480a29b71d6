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
// C = alpha * A^T * G without a transpose: a row of C is a column of A, and whoever owns it looks through A's columns and adds up the entries that are
// its own.  That reads nnz columns again and again, and takes one launch where transposition and product take seven: what a small training step costs
// is those launches.
//
// 32 vectors of kTransposedRows rows of C belong to `pieces` warps of a CTA, each of which looks through a run of A's entries; the pieces' sums are added
// in their order.  Runs have kTransposedRun entries as long as there are warps for them, and parts of rows are narrow, so that a column that holds all
// entries is neither one warp's to walk over nor one SM's to read.  (With a warp for a whole row, and a search and a wait for each entry, such a column
// took 0.32 us an entry: 640 us for 2048, where transposition and product take 18 to 27.)

constexpr int kTransposedThreads = 512;
constexpr int kTransposedRun = 128;
constexpr int kTransposedRows = 4;

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
    int log_pieces, run;  // entries of a piece, a multiple of 32
};

// A warp's entries among 128, in stored order: the row of G, the value and which of the warp's rows of C
struct OwnEntries {
    int row[kTransposedRun];
    float value[kTransposedRun];
    int of[kTransposedRun];
};

template <int VW>
__global__ void __launch_bounds__(kTransposedThreads, 2) spmm_transposed_kernel(TransposedParams p)
{
    constexpr int U = kTransposedRun / 32, W = kTransposedThreads / 32, R = kTransposedRows, kAtOnce = 4;
    __shared__ OwnEntries lists[W];
    __shared__ Vec<VW> sums[W][32];
    __shared__ bool any[W];
    wait_for_previous_grid();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int pieces = 1 << p.log_pieces, piece = warp & (pieces - 1);
    const long long own = ((long long)blockIdx.x * W + warp) >> p.log_pieces;  // rows of C and part of their columns
    const int parts = (p.nvec + 31) / 32;
    const long long row = own / parts * R;
    const int v = (int)(own % parts) * 32 + lane;
    const bool there = v < p.nvec;
    const float* const G = p.G + (long long)v * VW;
    const long long begin = (long long)piece * p.run, end = row < p.Kd ? min(begin + p.run, (long long)p.nnz) : 0;
    OwnEntries& list = lists[warp];
    Vec<VW> sum[R];
#pragma unroll
    for (int k = 0; k < R; ++k) sum[k].zero();
    bool found = false;
    for (long long base = begin; base < end; base += 32 * U) {
        int of[U];
        unsigned mine[U];
        int count = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long e = base + u * 32 + lane;
            of[u] = e < end ? (int)min(max(min(max(__ldg(p.col_idx + e), 0), p.Kd - 1) - row, -1LL), (long long)R) : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            mine[u] = __ballot_sync(kAllLanes, of[u] >= 0 && of[u] < R);
            count += __popc(mine[u]);
        }
        if (count == 0) continue;
        found = true;
        int r[U] = {};  // the last row that begins at the entry or before it
        if (count <= 2) {  // all lanes search for one: a step for five of a lane's own
#pragma unroll
            for (int u = 0; u < U; ++u) {
                for (unsigned left = mine[u]; left != 0; left &= left - 1) {
                    const int whose = __ffs(left) - 1, at = row_of_entry(p.row_ptr, p.M, (int)(base + u * 32) + whose, lane);
                    if (lane == whose) r[u] = at;
                }
            }
        } else {
            for (int length = p.M; length > 1; length -= length / 2) {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if ((mine[u] >> lane) & 1u && __ldg(p.row_ptr + r[u] + length / 2) <= (int)(base + u * 32 + lane)) r[u] += length / 2;
            }
        }
        int before = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if ((mine[u] >> lane) & 1u) {
                const int at = before + __popc(mine[u] & ((1u << lane) - 1u));
                list.row[at] = r[u];
                list.value[at] = __ldg(p.values + base + u * 32 + lane);
                list.of[at] = of[u];
            }
            before += __popc(mine[u]);
        }
        __syncwarp();
        for (int i0 = 0; i0 < count; i0 += kAtOnce) {
            Vec<VW> g[kAtOnce];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (i0 + i < count && there) g[i].load_nc(G + (long long)list.row[i0 + i] * p.ldg);
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                if (i0 + i < count && there) {
                    const float value = list.value[i0 + i];
                    const int k = list.of[i0 + i];
                    if (k == 0) sum[0].fma(value, g[i]);
                    else if (k == 1) sum[1].fma(value, g[i]);
                    else if (k == 2) sum[2].fma(value, g[i]);
                    else sum[3].fma(value, g[i]);
                }
            }
        }
        __syncwarp();
    }
    if (lane == 0) any[warp] = found;
    if (pieces > 1) __syncthreads();
#pragma unroll
    for (int k = 0; k < R; ++k) {
        if (pieces > 1) {
            if (piece != 0 && found) sums[warp][lane] = sum[k];
            __syncthreads();
            if (piece == 0) {
                for (int q = 1; q < pieces; ++q)
                    if (any[warp + q]) sum[k].fma(1.0f, sums[warp + q][lane]);
            }
            __syncthreads();
        }
        if (piece == 0 && row + k < p.Kd && there) sum[k].epilogue0(p.alpha).store(p.C + (row + k) * p.ldc + (long long)v * VW);
    }
}

}  // namespace csrspmm_b200

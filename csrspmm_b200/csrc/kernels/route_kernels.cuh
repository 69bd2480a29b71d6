// Routing: rows of dense scores -> a CSR matrix of k entries a row, and the gradient of the scores.
//
//     s = softmax(x) or sigmoid(x);  c = s + bias;  chosen: the k largest c among the top_groups best groups
//     w = scale * s / (sum of the chosen s)   or   scale * s
//
// The reference builds CSR matrices from dense ones by a threshold, on the host (src/host/csr_utils.cpp:70-116);
// there is no counterpart of a choice by rank.
//
// One warp owns a row and keeps it in registers, PER consecutive experts a lane, so that a row is read once and the
// lowest index among equals is the first lane's first element.  The choice has to be the one that scores in 64 bits
// make: fp32 scores tell two experts apart only where they differ by more than their rounding, so where the last one taken
// and the first one left out are nearer than that (kSigmoidMargin, kSoftmaxMargin), the warp makes the choice again in 64 bits.
// Without a bias the order of c is the order of x, and the choice is made on x itself, which tells apart what 64 bits round to the same
// (sigmoids of logits above 37, shares 745 below the largest); sums of two c that rank groups are in 64 bits.
#pragma once

#include <math_constants.h>

#include <type_traits>

#include "common.cuh"
#include "score_types.cuh"

namespace csrspmm_b200 {

constexpr int kRouteThreads = 256;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxChosen = 32;  // one lane each
constexpr int kRouteMaxGroups = 32;  // one lane each

// Twice what fp32 may be off in c, relative to max(1, |c|), in units of 2^-24.  Sigmoid: its slope is at most 1/4, and at most 0.224 / |x|, so that
// the exponential (4) and the rounding of its argument (2 |x|) make 1.5, the sum with 1, the reciprocal (2) and the sum with the bias 1, 2
// and 1: less than 8.  Softmax: the difference to the maximum, the argument (3 d exp(-d), d the difference), the exponential (4), the reciprocal (2),
// product, bias and the 5 steps of the sum across the warp make less than 16, its PER terms of a lane PER more.
constexpr float kUnit = 1.0f / 16777216.0f;
constexpr float kSigmoidMargin = 16.0f * kUnit, kSoftmaxMargin = 32.0f * kUnit;

struct RouteParams {
    int T, E, k;
    const void* x;
    long long ldx;
    const float* bias;  // may be null
    int groups, per_group, top_groups, group_top;
    int group_lanes, log_group_lanes;  // lanes of a group, a power of two, or 0
    int sigmoid, renormalize;
    float scale;
    int* row_ptr;
    int* col_idx;
    float* values;
};

struct RouteBackwardParams {
    int T, E, k;
    const void* x;
    long long ldx;
    const int* col_idx;
    const float* values;
    const float* dvalues;
    long long dv_stride;
    int sigmoid, renormalize;
    float scale;
    void* dx;
    long long ldd;
};

// PER experts of row `row` from `first` on; -infinity past the end
template <class T, int PER>
__device__ __forceinline__ void load_scores(const T* row, int E, int first, bool vectors, float (&x)[PER])
{
    constexpr int N = PER * sizeof(T) <= 16 ? PER : 16 / (int)sizeof(T);
    if (vectors) {
#pragma unroll
        for (int i = 0; i < PER; i += N) {
            if (first + i < E) {
                const Pack<T, N> v = *reinterpret_cast<const Pack<T, N>*>(row + first + i);
#pragma unroll
                for (int j = 0; j < N; ++j) x[i + j] = to_f32(v.v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) x[i + j] = -CUDART_INF_F;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) x[i] = first + i < E ? to_f32(row[first + i]) : -CUDART_INF_F;
    }
}

template <class T, int PER>
__device__ __forceinline__ bool whole_vectors(const void* x, long long ld, int E)
{
    constexpr int N = PER * sizeof(T) <= 16 ? PER : 16 / (int)sizeof(T);
    return E % N == 0 && ld % N == 0 && (reinterpret_cast<uintptr_t>(x) & (N * sizeof(T) - 1)) == 0;
}

// The largest group_top of each group, summed, by the lane whose number the group has (lanes beyond: -infinity); c by expert in `row`.  *size: how
// large what was summed is, for the bound of its rounding.
template <class F>
__device__ __forceinline__ F group_score(const RouteParams& p, const F* row, int lane, F* size)
{
    F score = (F)-CUDART_INF_F;
    *size = 0;
    if (lane < p.groups) {
        F best = (F)-CUDART_INF_F, second = (F)-CUDART_INF_F;
        int at = lane % p.per_group;  // lanes begin at different banks
#pragma unroll 4
        for (int j = 0; j < p.per_group; ++j) {
            const F v = row[lane * p.per_group + at];
            if (v > best) second = best, best = v;
            else if (v > second) second = v;
            if (++at == p.per_group) at = 0;
        }
        score = p.group_top == 2 ? best + second : best;
        *size = (best < -1 || best > 1 ? fabs(best) : 1) + (p.group_top == 2 ? second < -1 || second > 1 ? fabs(second) : 1 : 0);
    }
    return score == score ? score : (F)-CUDART_INF_F;  // -infinity and +infinity
}

// Whether group `mine` is among the best, of which `of_group(g)` gives each one's score.
template <class F, class G>
__device__ __forceinline__ bool among_best(const RouteParams& p, F score, int mine, G&& of_group)
{
    int rank = 0;
    for (int g = 0; g < p.groups; ++g) {
        const F other = of_group(g);
        rank += other > score || (other == score && g < mine);
    }
    return mine < p.groups && rank < p.top_groups;
}

// Descending, by Batcher's odd-even merges
template <int N>
__device__ __forceinline__ void sort_descending(float (&v)[N])
{
#pragma unroll
    for (int run = 1; run < N; run *= 2) {
#pragma unroll
        for (int k = run; k >= 1; k /= 2) {
#pragma unroll
            for (int j = k % run; j + k < N; j += 2 * k) {
#pragma unroll
                for (int i = 0; i < k; ++i) {
                    if (i + j + k < N && (i + j) / (2 * run) == (i + j + k) / (2 * run)) {
                        const float high = fmaxf(v[i + j], v[i + j + k]);
                        v[i + j + k] = fminf(v[i + j], v[i + j + k]);
                        v[i + j] = high;
                    }
                }
            }
        }
    }
}

// exp(v), off by 2^-22 and by the rounding of v log2(e): enough for a choice that is checked
__device__ __forceinline__ float exp_near(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * CUDART_L2E_F));
    return r;
}
__device__ __forceinline__ float reciprocal_near(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Which of this lane's experts are in a group that is kept, as bits.  *near: exact sums may keep another one.  margin (negative: the order is exact): as
// for two c.  A group's sum may be off by half of that for each c in it, relative to max(1, |c|) of that c and not to the sum, in which a bias of
// 10000 and one of -10000 leave nothing of their size; the constants leave room for the rounding of the sum itself.
template <int PER>
__device__ __forceinline__ unsigned open_groups(const RouteParams& p, const float (&c)[PER], int lane, float* row, float margin, bool* near)
{
    const int first = lane * PER;
    float score, size;
    bool kept, there;
    unsigned open = 0;
    if (p.group_lanes > 0) {  // a group is that many lanes, a power of two
        float best = c[0], second = -CUDART_INF_F;
#pragma unroll
        for (int i = 1; i < PER; ++i) {
            second = fmaxf(second, fminf(best, c[i]));
            best = fmaxf(best, c[i]);
        }
        for (int d = 1; d < p.group_lanes; d *= 2) {
            const float other = __shfl_xor_sync(kAllLanes, best, d), behind = __shfl_xor_sync(kAllLanes, second, d);
            second = fmaxf(fmaxf(second, behind), fminf(best, other));
            best = fmaxf(best, other);
        }
        score = p.group_top == 2 ? best + second : best;
        score = score == score ? score : -CUDART_INF_F;  // -infinity and +infinity
        size = fmaxf(1.0f, fabsf(best)) + (p.group_top == 2 ? fmaxf(1.0f, fabsf(second)) : 0.0f);
        const int mine = lane >> p.log_group_lanes;
        there = mine < p.groups;
        kept = among_best(p, score, mine, [&](int g) { return __shfl_sync(kAllLanes, score, g << p.log_group_lanes); });
        open = kept ? kAllLanes : 0u;
    } else {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (first + i < p.E) row[first + i] = c[i];
        __syncwarp();
        score = group_score(p, row, lane, &size);
        there = lane < p.groups;
        kept = among_best(p, score, lane, [&](int g) { return __shfl_sync(kAllLanes, score, g); });
        const unsigned groups = __ballot_sync(kAllLanes, kept);
        int g = first / p.per_group, left = p.per_group - (first - g * p.per_group);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            open |= ((groups >> (g & 31)) & 1u) << i;
            if (--left == 0) ++g, left = p.per_group;
        }
    }
    if (margin >= 0.0f) {
        // the least that a kept one may be and the most that one left out may be; without a number (infinities of both signs): left out of this
        const float off = 0.5f * margin * size;
        const float last = -warp_max(kept ? off - score : -CUDART_INF_F), next = warp_max(there && !kept ? score + off : -CUDART_INF_F);
        if (next > -CUDART_INF_F && last <= next) *near = true;
    }
    return open;
}

__device__ __forceinline__ float sigmoid_of(float x) { return 1.0f / (1.0f + expf(-x)); }

// exp(v) in 64 bits for v <= 0, to a unit or two, without a branch: exp(v) = 2^n exp(r) with |r| <= ln(2) / 2, and the series of exp up to r^13 / 13!,
// behind which less than 1e-17 follows.  (The library's has branches: eight of them, one behind the other, were most of 6 us that one
// row in some thousands took longer than the others, which a launch then waited for.)
__device__ __forceinline__ double exp_of_negative(double v)
{
    v = v > -1400.0 ? v : -1400.0;
    const double n = rint(v * 1.4426950408889634);
    double r = fma(n, -0.69314718055994529, v);
    r = fma(n, -2.3190468138462996e-17, r);  // ln(2) less the double above
    double e = 1.0 / 6227020800.0;
    constexpr double kOneOver[13] = {1.0 / 479001600, 1.0 / 39916800, 1.0 / 3628800, 1.0 / 362880, 1.0 / 40320, 1.0 / 5040, 1.0 / 720,
                                     1.0 / 120,       1.0 / 24,       1.0 / 6,       0.5,          1.0,         1.0};
#pragma unroll
    for (int i = 0; i < 13; ++i) e = fma(e, r, kOneOver[i]);
    const int half = (int)n / 2, rest = (int)n - half;  // two factors: the result may be below the normal numbers
    return e * __hiloint2double((1023 + half) << 20, 0) * __hiloint2double((1023 + rest) << 20, 0);
}

// 1 / v in 64 bits for 1 <= v < 2^20: fp32's, and Newton's step three times
__device__ __forceinline__ double reciprocal(double v)
{
    double r = (double)reciprocal_near((float)v);
#pragma unroll
    for (int i = 0; i < 3; ++i) r = fma(r, fma(-v, r, 1.0), r);
    return r;
}

// The experts a row takes, as bits of the lane that holds them; the choice is made on c in fp32 or, with ON_X and within groups that are ranked by sums,
// on the logits, whose order is that of c where there is no bias.  *near: in 64 bits the choice may be another one.
//
// Every lane sorts its experts' c; the largest heads of the lanes are taken off until k are, which gives the last c taken, and the experts
// are those above it and as many at it as are left, in the order of their numbers.  That takes 19 instructions a round where marking
// the largest of all in each round took 60.
template <int PER, bool ON_X>
__device__ __forceinline__ unsigned choose(const RouteParams& p, const float (&x)[PER], int lane, float* row, bool* near)
{
    const int first = lane * PER;
    const float margin = p.sigmoid ? kSigmoidMargin : kSoftmaxMargin + 2.0f * PER * kUnit;
    float c[PER];
    if constexpr (ON_X) {
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] = x[i];
    } else {
        if (p.sigmoid) {
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] = reciprocal_near(1.0f + exp_near(-x[i]));
        } else {
            float m = x[0];
#pragma unroll
            for (int i = 1; i < PER; ++i) m = fmaxf(m, x[i]);
            m = warp_max(m);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                c[i] = x[i] > -CUDART_INF_F ? exp_near(x[i] - m) : 0.0f;
                sum += c[i];
            }
            sum = reciprocal_near(warp_sum(sum));
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] *= sum;
        }
        if (p.bias != nullptr) {
            float bias[PER];
            load_scores<float, PER>(p.bias, p.E, first, whole_vectors<float, PER>(p.bias, 0, p.E), bias);
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] += bias[i];
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) c[i] = x[i] > -CUDART_INF_F && c[i] > -CUDART_INF_F ? c[i] : -CUDART_INF_F;  // not available, or NaN
    unsigned open = kAllLanes;
    if (p.top_groups < p.groups) {
        open = open_groups<PER>(p, c, lane, row, ON_X ? -1.0f : margin, near);
        if constexpr (!ON_X) {
            if (p.bias == nullptr) {
#pragma unroll
                for (int i = 0; i < PER; ++i) c[i] = x[i] > -CUDART_INF_F ? x[i] : -CUDART_INF_F;
            }
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] = (open >> i) & 1u ? c[i] : -CUDART_INF_F;
    }

    float head[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) head[i] = c[i];
    sort_descending(head);
    int count = 0;
    float last;
    do {
        last = warp_max(head[0]);
        const bool off = head[0] == last;
        count += __popc(__ballot_sync(kAllLanes, off));
        if (off) {
#pragma unroll
            for (int i = 0; i + 1 < PER; ++i) head[i] = head[i + 1];
            head[PER - 1] = -CUDART_INF_F;
        }
    } while (count < p.k && last > -CUDART_INF_F);
    unsigned taken = 0;
    if (last > -CUDART_INF_F) {
        const float next = warp_max(head[0]);  // of those that were not taken off: at `last` itself there may be more
        if constexpr (!ON_X) {
            if (p.bias != nullptr && (count > p.k || (next > -CUDART_INF_F && last - next <= margin * fmaxf(1.0f, fabsf(last))))) *near = true;
        }
        if (count == p.k && next < last) {
#pragma unroll
            for (int i = 0; i < PER; ++i) taken |= (unsigned)(c[i] >= last) << i;
            return taken;
        }
    }
    unsigned at = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        taken |= (unsigned)(c[i] > last) << i;
        at |= (unsigned)(c[i] == last && (last > -CUDART_INF_F || (((open >> i) & 1u) && first + i < p.E))) << i;  // fewer than k available: any of the open
    }
    const int wanted = p.k - (int)__reduce_add_sync(kAllLanes, (unsigned)__popc(taken));
    int before = __popc(at);  // the lowest numbers
    const int own = before;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(kAllLanes, before, d);
        if (lane >= d) before += v;
    }
    before -= own;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if ((at >> i) & 1u) {
            if (before < wanted) taken |= 1u << i;
            ++before;
        }
    }
    return taken;
}

// The same in 64 bits, on c in shared memory.  Few rows come here (2 to 4 of 16384 with 256 experts), and what counts is that the others do not
// pay for it: as an inlined copy of the code above, or as a function of its own, it cost every row half as much again in registers.
template <class T, int PER>
__device__ __forceinline__ unsigned choose_exactly(const RouteParams& p, const T* scores, int lane, double* row)
{
    float m = -CUDART_INF_F;
    double sum = 0.0;
    if (!p.sigmoid) {
#pragma unroll 1
        for (int e = lane; e < p.E; e += 32) m = fmaxf(m, to_f32(scores[e]));
        m = warp_max(m);
#pragma unroll 1
        for (int e = lane; e < p.E; e += 32) {
            const float x = to_f32(scores[e]);
            if (x > -CUDART_INF_F) sum += exp_of_negative((double)x - (double)m);
        }
        sum = reciprocal(warp_sum(sum));
    }
    __syncwarp();
#pragma unroll 2
    for (int e = lane; e < p.E; e += 32) {
        const float x = to_f32(scores[e]);
        const double t = exp_of_negative(p.sigmoid ? -fabs((double)x) : (double)x - (double)m);
        double c = p.sigmoid ? (x < 0.0f ? t : 1.0) * reciprocal(1.0 + t) : t * sum;
        if (p.bias != nullptr) c += (double)__ldg(p.bias + e);
        row[e] = x > -CUDART_INF_F && c > -CUDART_INF ? c : -CUDART_INF;
    }
    __syncwarp();
    if (p.top_groups < p.groups) {
        double size;
        const double score = group_score(p, row, lane, &size);
        const unsigned kept = __ballot_sync(kAllLanes, among_best(p, score, lane, [&](int g) { return __shfl_sync(kAllLanes, score, g); }));
        __syncwarp();
#pragma unroll 1
        for (int e = lane; e < p.E; e += 32)
            if (!((kept >> (e / p.per_group)) & 1u)) row[e] = CUDART_NAN;
        if (p.bias == nullptr) {
#pragma unroll 1
            for (int e = lane; e < p.E; e += 32) {
                const float x = to_f32(scores[e]);
                if (row[e] == row[e]) row[e] = x > -CUDART_INF_F ? (double)x : -CUDART_INF;
            }
        }
    }
    unsigned taken = 0;
#pragma unroll 1
    for (int r = 0; r < p.k; ++r) {  // the largest, of equals the lowest number
        double best = 0.0;
        int which = -1;
#pragma unroll 4
        for (int e = lane; e < p.E; e += 32) {
            const double c = row[e];
            if (c == c && (which < 0 || c > best)) best = c, which = e;
        }
        unsigned long long key = (unsigned long long)__double_as_longlong(best);  // in the order of the numbers; 0: none
        key = which < 0 ? 0 : (key >> 63) ? ~key : (key | 0x8000000000000000ull);
        const unsigned high = __reduce_max_sync(kAllLanes, (unsigned)(key >> 32));
        const unsigned low = __reduce_max_sync(kAllLanes, (unsigned)(key >> 32) == high ? (unsigned)key : 0u);
        const bool has = which >= 0 && key == (((unsigned long long)high << 32) | low);
        const int e = (int)__reduce_min_sync(kAllLanes, has ? (unsigned)which : 0x7fffffffu);
        if (e == which) row[e] = CUDART_NAN;
        if (e / PER == lane) taken |= 1u << (e % PER);
    }
    return taken;
}

template <class T, int PER, bool ON_X>
__global__ void __launch_bounds__(kRouteThreads, PER <= 8 ? 5 : PER == 16 ? 4 : 2) route_kernel(RouteParams p)
{
    // a row of c, in doubles where the choice is made again
    extern __shared__ __align__(16) char route_smem[];
    wait_for_previous_grid();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = (long long)blockIdx.x * (kRouteThreads / 32) + warp;
    if (row >= p.T) return;
    __shared__ int chosen_at[kRouteThreads / 32][kRouteMaxChosen];
    double* const row_smem = reinterpret_cast<double*>(route_smem) + (size_t)warp * p.E;

    float x[PER];
    const T* const scores = static_cast<const T*>(p.x) + row * p.ldx;
    load_scores<T, PER>(scores, p.E, lane * PER, whole_vectors<T, PER>(p.x, p.ldx, p.E), x);
    bool near = false;
    unsigned taken = choose<PER, ON_X>(p, x, lane, reinterpret_cast<float*>(row_smem), &near);
    if constexpr (!ON_X) {
        if (__any_sync(kAllLanes, near)) taken = choose_exactly<T, PER>(p, scores, lane, row_smem);
    }

    // ascending columns: lanes hold ascending runs
    int before = __popc(taken);
    const int own = before;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(kAllLanes, before, d);
        if (lane >= d) before += v;
    }
    bool broken = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) broken |= x[i] != x[i] || (!p.sigmoid && x[i] == CUDART_INF_F);
    broken = __any_sync(kAllLanes, broken);
    for (int at = before - own; taken != 0 && at < kRouteMaxChosen; ++at) {
        chosen_at[warp][at] = lane * PER + __ffs(taken) - 1;
        taken &= taken - 1;
    }
    __syncwarp();
    const bool mine = lane < p.k;
    const int col = mine ? chosen_at[warp][lane] : 0;
    const float v = mine ? to_f32(scores[col]) : -CUDART_INF_F;
    float w;
    if (p.renormalize) {  // shares of the chosen, scaled so that their sum does not vanish: t = s * exp(-m)
        float m = warp_max(v);
        float t = 0.0f;
        if (v > -CUDART_INF_F) {
            if (p.sigmoid) {
                m = fminf(m, 0.0f);
                t = expf(fminf(v, 0.0f) - m) / (1.0f + expf(-fabsf(v)));
            } else {
                t = expf(v - m);
            }
        }
        const float sum = warp_sum(t);
        w = sum > 0.0f ? t / sum : 0.0f;
    } else if (p.sigmoid) {
        w = sigmoid_of(v);
    } else {
        float m = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < PER; ++i) m = fmaxf(m, x[i]);
        m = warp_max(m);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) sum += x[i] > -CUDART_INF_F ? expf(x[i] - m) : 0.0f;
        sum = warp_sum(sum);
        w = v > -CUDART_INF_F ? expf(v - m) / sum : 0.0f;
    }
    w *= p.scale;
    if (broken) w = CUDART_NAN_F;
    if (mine) {
        p.col_idx[row * p.k + lane] = col;
        p.values[row * p.k + lane] = w;
    }
    if (lane == 0) p.row_ptr[row] = (int)(row * p.k);
    if (lane == 0 && row == p.T - 1) p.row_ptr[p.T] = p.T * p.k;
}

// With p = w / scale:
//     softmax, renormalised      dx_j = w_j (g_j - sum p g)             for the chosen, 0 elsewhere
//     sigmoid, renormalised      dx_j = w_j (1 - s_j) (g_j - sum p g)
//     sigmoid                    dx_j = w_j (1 - s_j) g_j
//     softmax                    dx_i = s_i (scale g_i [chosen] - sum w g)
template <class T, int PER>
__global__ void __launch_bounds__(kRouteThreads) route_backward_kernel(RouteBackwardParams p)
{
    wait_for_previous_grid();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = (long long)blockIdx.x * (kRouteThreads / 32) + warp;
    if (row >= p.T) return;
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    T* dx = static_cast<T*>(p.dx) + row * p.ldd;
    const bool mine = lane < p.k;
    int col = 0;
    float w = 0.0f, g = 0.0f;
    if (mine) {
        col = min(max(p.col_idx[row * p.k + lane], 0), p.E - 1);
        w = p.values[row * p.k + lane];
        g = p.dvalues[(row * p.k + lane) * p.dv_stride];
    }
    const bool broken = __any_sync(kAllLanes, w != w);
    float at_chosen, elsewhere[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) elsewhere[i] = 0.0f;
    if (p.sigmoid || p.renormalize) {
        float away = g;
        if (p.renormalize) away -= warp_sum(p.scale != 0.0f ? w / p.scale * g : 0.0f);
        at_chosen = w * away;
        if (p.sigmoid && mine) at_chosen *= 1.0f / (1.0f + expf(to_f32(x[col])));  // 1 - s
    } else {
        float s[PER];
        load_scores<T, PER>(x, p.E, lane * PER, whole_vectors<T, PER>(p.x, p.ldx, p.E), s);
        float m = -CUDART_INF_F;
#pragma unroll
        for (int i = 0; i < PER; ++i) m = fmaxf(m, s[i]);
        m = warp_max(m);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            s[i] = s[i] > -CUDART_INF_F ? expf(s[i] - m) : 0.0f;
            sum += s[i];
        }
        sum = warp_sum(sum);
        const float mean = warp_sum(w * g);
#pragma unroll
        for (int i = 0; i < PER; ++i) elsewhere[i] = sum > 0.0f ? -(s[i] / sum) * mean : 0.0f;
        const float own = mine ? to_f32(x[col]) : -CUDART_INF_F;
        at_chosen = own > -CUDART_INF_F ? expf(own - m) / sum * (p.scale * g - mean) : 0.0f;
    }
    if (broken) {
        at_chosen = CUDART_NAN_F;
#pragma unroll
        for (int i = 0; i < PER; ++i) elsewhere[i] = CUDART_NAN_F;
    }
    constexpr int N = PER * sizeof(T) <= 16 ? PER : 16 / (int)sizeof(T);
    const int first = lane * PER;
    if (whole_vectors<T, PER>(p.dx, p.ldd, p.E)) {
#pragma unroll
        for (int i = 0; i < PER; i += N) {
            if (first + i < p.E) {
                Pack<T, N> v;
#pragma unroll
                for (int j = 0; j < N; ++j) v.v[j] = from_f32<T>(elsewhere[i + j]);
                *reinterpret_cast<Pack<T, N>*>(dx + first + i) = v;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (first + i < p.E) dx[first + i] = from_f32<T>(elsewhere[i]);
    }
    __syncwarp();  // the chosen are written over it, after it
    if (mine) dx[col] = from_f32<T>(at_chosen);
}

}  // namespace csrspmm_b200

// Routing: rows of dense scores -> a CSR matrix of k entries a row, and the gradient of the scores.
//
//     s = softmax(x) or sigmoid(x);  c = s + bias;  chosen: the k largest c among the top_groups best groups
//     w = scale * s / (sum of the chosen s)   or   scale * s
//
// The reference builds CSR matrices from dense ones by a threshold, on the host (src/host/csr_utils.cpp:70-116);
// there is no counterpart of a choice by rank.
//
// One warp owns a row and keeps it in registers, PER consecutive experts a lane, so that a row is read once and the
// lowest index among equals is the first lane's first element.  The choice has to be the one that exact arithmetic
// makes: fp32 scores tell two experts apart only where they differ by more than their rounding, so where the last one taken
// and the first one left out are nearer than that (kChoiceMargin), the warp makes the choice again in 64 bits.
// Without a bias the order of c is the order of x, and the choice is made on x itself.
#pragma once

#include <math_constants.h>

#include "common.cuh"
#include "score_types.cuh"

namespace csrspmm_b200 {

constexpr int kRouteThreads = 256;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxChosen = 32;  // one lane each
constexpr int kRouteMaxGroups = 32;  // one lane each

// Twice what fp32 may be off in c, relative to max(1, |c|): s is below 1, and the difference to the maximum (less than one unit of
// 2^-24, as d exp(-d) is), the exponential (2), the sum (32 terms of a lane and 5 steps across the warp, 37), the division and
// the sum with the bias (1 each, and 1 for the product) round it by less than 64 units together.
constexpr float kChoiceMargin = 128.0f / 16777216.0f;

struct RouteParams {
    int T, E, k;
    const void* x;
    long long ldx;
    const float* bias;  // may be null
    int groups, per_group, top_groups, group_top;
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

// Keys in the order of the numbers they stand for; kNotThere < kNotAvailable < everything else.
__device__ __forceinline__ unsigned order_key(float c)
{
    const unsigned u = __float_as_uint(c);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ unsigned long long order_key(double c)
{
    const unsigned long long u = (unsigned long long)__double_as_longlong(c);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
constexpr unsigned kNotThere = 0, kNotAvailable = 1;

__device__ __forceinline__ float key_value(unsigned key)
{
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

__device__ __forceinline__ unsigned warp_max_key(unsigned v) { return __reduce_max_sync(kAllLanes, v); }
__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long v)
{
    const unsigned hi = __reduce_max_sync(kAllLanes, (unsigned)(v >> 32));
    const unsigned lo = __reduce_max_sync(kAllLanes, (unsigned)(v >> 32) == hi ? (unsigned)v : 0u);
    return ((unsigned long long)hi << 32) | lo;
}

template <class F>
struct KeyOf;
template <>
struct KeyOf<float> {
    using type = unsigned;
};
template <>
struct KeyOf<double> {
    using type = unsigned long long;
};

__device__ __forceinline__ float exponential(float v) { return expf(v); }
__device__ __forceinline__ double exponential(double v) { return exp(v); }

// The experts a row takes, as bits of the lane that holds them.  F: the type the choice is made in.  ON_X: c is ordered as x is.
// *near: the choice may be another one in exact arithmetic (never set for doubles).
template <class F, int PER, bool ON_X>
__device__ __forceinline__ unsigned choose(const RouteParams& p, const float (&x)[PER], int lane, float* group_smem, bool* near)
{
    using Key = typename KeyOf<F>::type;
    const int first = lane * PER;
    F c[PER];
    if constexpr (ON_X) {
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] = (F)x[i];
    } else {
        if (p.sigmoid) {
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] = (F)1 / ((F)1 + exponential(-(F)x[i]));
        } else {
            float m = -CUDART_INF_F;
#pragma unroll
            for (int i = 0; i < PER; ++i) m = fmaxf(m, x[i]);
            m = warp_max(m);
            F sum = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                c[i] = x[i] > -CUDART_INF_F ? exponential((F)x[i] - (F)m) : (F)0;
                sum += c[i];
            }
            sum = warp_sum(sum);
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] = c[i] / sum;
        }
        if (p.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (first + i < p.E) c[i] += (F)__ldg(p.bias + first + i);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (!(x[i] > -CUDART_INF_F)) c[i] = (F)-CUDART_INF_F;  // -infinity and NaN
    }

    unsigned kept = kAllLanes;  // groups
    if (p.top_groups < p.groups) {
        F* row = reinterpret_cast<F*>(group_smem);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (first + i < p.E) row[first + i] = c[i];
        __syncwarp();
        F score = (F)-CUDART_INF_F;
        if (lane < p.groups) {
            F best = (F)-CUDART_INF_F, second = (F)-CUDART_INF_F;
            for (int j = 0; j < p.per_group; ++j) {
                int at = j + lane;  // lanes begin at different banks
                at = at < p.per_group ? at : at % p.per_group;
                const F v = row[lane * p.per_group + at];
                if (v > best) second = best, best = v;
                else if (v > second) second = v;
            }
            score = p.group_top == 2 ? best + second : best;
            if (score != score) score = (F)-CUDART_INF_F;
        }
        int rank = 0;
        for (int g = 0; g < p.groups; ++g) {
            const F other = __shfl_sync(kAllLanes, score, g);
            rank += other > score || (other == score && g < lane);
        }
        const bool mine = lane < p.groups && rank < p.top_groups;
        kept = __ballot_sync(kAllLanes, mine);
        if constexpr (sizeof(F) == 4 && !ON_X) {
            const Key worst_in = ~warp_max_key(~(mine ? order_key(score) : ~(Key)0));
            const Key best_out = warp_max_key(lane < p.groups && !mine ? order_key(score) : (Key)0);
            const float a = key_value(worst_in), b = key_value(best_out);
            if (b > -CUDART_INF_F && a - b <= 2.0f * kChoiceMargin * fmaxf(1.0f, fabsf(a))) *near = true;
        }
    }

    Key key[PER];
    int g = first / p.per_group, left = p.per_group - (first - g * p.per_group);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const bool there = first + i < p.E && ((kept >> (g & 31)) & 1u);
        key[i] = !there ? (Key)kNotThere : c[i] > (F)-CUDART_INF_F ? order_key(c[i]) : (Key)kNotAvailable;
        if (--left == 0) ++g, left = p.per_group;
    }
    unsigned taken = 0;
    Key last = 0;
    for (int r = 0; r < p.k; ++r) {
        Key mine = key[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) mine = key[i] > mine ? key[i] : mine;
        last = warp_max_key(mine);
        const unsigned holders = __ballot_sync(kAllLanes, mine == last);
        if (lane == __ffs(holders) - 1) {
            bool done = false;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (!done && key[i] == last) key[i] = (Key)kNotThere, taken |= 1u << i, done = true;
        }
    }
    if constexpr (sizeof(F) == 4 && !ON_X) {
        Key mine = key[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) mine = key[i] > mine ? key[i] : mine;
        const Key next = warp_max_key(mine);
        if (next > kNotAvailable) {  // then so is the last one taken
            const float a = key_value(last), b = key_value(next);
            if (a - b <= kChoiceMargin * fmaxf(1.0f, fabsf(a))) *near = true;
        }
    }
    return taken;
}

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

__device__ __forceinline__ float sigmoid_of(float x) { return 1.0f / (1.0f + expf(-x)); }

template <class T, int PER, bool ON_X>
__global__ void __launch_bounds__(kRouteThreads) route_kernel(RouteParams p)
{
    // a row of c where groups are ranked (doubles where the choice is made again), then the chosen: index and score
    extern __shared__ __align__(16) char route_smem[];
    wait_for_previous_grid();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = (long long)blockIdx.x * (kRouteThreads / 32) + warp;
    if (row >= p.T) return;
    __shared__ int chosen_at[kRouteThreads / 32][kRouteMaxChosen];
    __shared__ float chosen_x[kRouteThreads / 32][kRouteMaxChosen];
    float* group_smem = reinterpret_cast<float*>(route_smem) + (size_t)warp * 2 * p.E;

    float x[PER];
    load_scores<T, PER>(static_cast<const T*>(p.x) + row * p.ldx, p.E, lane * PER, whole_vectors<T, PER>(p.x, p.ldx, p.E), x);
    bool near = false;
    unsigned taken = choose<float, PER, ON_X>(p, x, lane, group_smem, &near);
    if constexpr (!ON_X) {
        if (__any_sync(kAllLanes, near)) taken = choose<double, PER, ON_X>(p, x, lane, group_smem, &near);
    }

    // ascending columns: lanes hold ascending runs
    int before = __popc(taken);
    const int own = before;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(kAllLanes, before, d);
        if (lane >= d) before += v;
    }
    int at = before - own;
    bool broken = false;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if ((taken >> i) & 1u) {
            chosen_at[warp][at] = lane * PER + i;
            chosen_x[warp][at] = x[i];
            ++at;
        }
        broken |= x[i] != x[i] || (!p.sigmoid && x[i] == CUDART_INF_F);
    }
    broken = __any_sync(kAllLanes, broken);
    __syncwarp();
    const bool mine = lane < p.k;
    const float v = mine ? chosen_x[warp][lane] : -CUDART_INF_F;
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
        p.col_idx[row * p.k + lane] = chosen_at[warp][lane];
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

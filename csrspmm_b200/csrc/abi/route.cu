// extern "C" entry points for routing (declared in include/csrspmm_b200.h): dense scores -> CSR matrix by rank, and the
// gradient of the scores.  The reference makes CSR matrices from dense ones by a threshold only
// (src/host/csr_utils.cpp:70-116).
#include <cuda_runtime.h>

#include <cmath>
#include <type_traits>

#include "../kernels/route_kernels.cuh"
#include "csrspmm_b200.h"
#include "pdl.h"
#include "plan.h"

using namespace csrspmm_b200;

#define CUDA_TRY(expr)                                                                        \
    do {                                                                                      \
        cudaError_t e__ = (expr);                                                             \
        if (e__ != cudaSuccess) {                                                             \
            set_last_error("%s failed: %s (%s:%d)", #expr, cudaGetErrorString(e__), __FILE__, \
                           __LINE__);                                                         \
            return CSRSPMM_B200_ERR_CUDA;                                                     \
        }                                                                                     \
    } while (0)

namespace {

int refuse(const char* what)
{
    set_last_error("route: %s", what);
    return CSRSPMM_B200_ERR_BAD_ARG;
}

int check(const csrspmm_b200_route_args* a)
{
    if (a == nullptr || a->struct_size != sizeof(csrspmm_b200_route_args)) return refuse("args is null or args.struct_size wrong");
    if (a->T < 0 || a->E < 1 || a->E > kRouteMaxExperts) return refuse("needs rows and 1 to 1024 experts");
    if (a->score_type < CSRSPMM_B200_F32 || a->score_type > CSRSPMM_B200_BF16) return refuse("unknown score_type");
    if (a->score != CSRSPMM_B200_SOFTMAX && a->score != CSRSPMM_B200_SIGMOID) return refuse("unknown score");
    if (a->groups < 1 || a->groups > kRouteMaxGroups || a->E % a->groups != 0) return refuse("groups has to divide E and be 1 to 32");
    if (a->top_groups < 1 || a->top_groups > a->groups) return refuse("top_groups has to be 1 to groups");
    if (a->group_top < 1 || a->group_top > 2 || a->group_top > a->E / a->groups) return refuse("group_top has to be 1 or 2 and no more than a group holds");
    if (a->k < 1 || a->k > kRouteMaxChosen || a->k > a->top_groups * (a->E / a->groups))
        return refuse("k has to be 1 to 32 and no more than the groups taken hold");
    if ((long long)a->T * a->k > 0x7fffffffLL) return refuse("more than 2^31 - 1 entries");
    if (a->ld < a->E) return refuse("ld is less than E");
    if (!std::isfinite(a->scale)) return refuse("scale has to be finite");
    if (a->T > 0 && a->scores == nullptr) return refuse("scores is null");
    return CSRSPMM_B200_OK;
}

// f(type, experts per lane) for the types and sizes of these arguments
template <class F>
cudaError_t for_shape(const csrspmm_b200_route_args* a, F&& f)
{
    auto with_type = [&](auto zero) -> cudaError_t {
        using T = decltype(zero);
        if (a->E <= 64) return f(zero, std::integral_constant<int, 2>());
        if (a->E <= 128) return f(zero, std::integral_constant<int, 4>());
        if (a->E <= 256) return f(zero, std::integral_constant<int, 8>());
        if (a->E <= 512) return f(zero, std::integral_constant<int, 16>());
        return f(zero, std::integral_constant<int, 32>());
    };
    if (a->score_type == CSRSPMM_B200_F32) return with_type(float());
    if (a->score_type == CSRSPMM_B200_F16) return with_type(__half());
    return with_type(__nv_bfloat16());
}

unsigned grid_of(int32_t T) { return (unsigned)(((long long)T + kRouteThreads / 32 - 1) / (kRouteThreads / 32)); }

}  // namespace

extern "C" {

int csrspmm_b200_route(const csrspmm_b200_route_args* a, int32_t* row_ptr, int32_t* col_idx, float* values, csrspmm_b200_stream_t stream)
{
    if (const int bad = check(a)) return bad;
    if (row_ptr == nullptr || (a->T > 0 && (col_idx == nullptr || values == nullptr))) return refuse("null pointer");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a->T == 0) {
        CUDA_TRY(cudaMemsetAsync(row_ptr, 0, sizeof(int32_t), st));
        return CSRSPMM_B200_OK;
    }
    RouteParams p = {};
    p.T = a->T, p.E = a->E, p.k = a->k;
    p.x = a->scores, p.ldx = a->ld, p.bias = a->bias;
    p.groups = a->groups, p.per_group = a->E / a->groups, p.top_groups = a->top_groups, p.group_top = a->group_top;
    p.sigmoid = a->score == CSRSPMM_B200_SIGMOID, p.renormalize = a->renormalize, p.scale = a->scale;
    p.row_ptr = row_ptr, p.col_idx = col_idx, p.values = values;
    const bool ranks_groups = a->top_groups < a->groups;
    const bool on_x = a->bias == nullptr && (!ranks_groups || a->group_top == 1);
    const size_t smem = ranks_groups || !on_x ? (size_t)(kRouteThreads / 32) * 8 * (size_t)a->E : 0;
    CUDA_TRY(for_shape(a, [&](auto zero, auto per) {
        constexpr int per_lane = decltype(per)::value;
        const int lanes = p.per_group % per_lane == 0 ? p.per_group / per_lane : 0;
        for (p.log_group_lanes = 0; 1 << p.log_group_lanes < lanes;) ++p.log_group_lanes;
        p.group_lanes = lanes > 0 && 1 << p.log_group_lanes == lanes ? lanes : 0;
        auto launch = [&](auto x_c) {
            constexpr auto kernel = route_kernel<decltype(zero), per_lane, decltype(x_c)::value>;
            if (smem > 40 * 1024) {  // 48 KB without asking, the kernel's own 1 KB among them
                const cudaError_t e = allow_dynamic_smem<kernel>(smem);
                if (e != cudaSuccess) return e;
            }
            return launch_overlapped(kernel, grid_of(a->T), kRouteThreads, smem, st, p);
        };
        return on_x ? launch(std::true_type()) : launch(std::false_type());
    }));
    return CSRSPMM_B200_OK;
}

int csrspmm_b200_route_backward(const csrspmm_b200_route_args* a, const int32_t* col_idx, const float* values, const float* dvalues,
                                int64_t dvalues_stride, void* dscores, int64_t ldd, csrspmm_b200_stream_t stream)
{
    if (const int bad = check(a)) return bad;
    if (ldd < a->E) return refuse("ldd is less than E");
    if (a->T == 0) return CSRSPMM_B200_OK;
    if (col_idx == nullptr || values == nullptr || dvalues == nullptr || dscores == nullptr) return refuse("null pointer");
    RouteBackwardParams p = {};
    p.T = a->T, p.E = a->E, p.k = a->k;
    p.x = a->scores, p.ldx = a->ld;
    p.col_idx = col_idx, p.values = values, p.dvalues = dvalues, p.dv_stride = dvalues_stride;
    p.sigmoid = a->score == CSRSPMM_B200_SIGMOID, p.renormalize = a->renormalize, p.scale = a->scale;
    p.dx = dscores, p.ldd = ldd;
    CUDA_TRY(for_shape(a, [&](auto zero, auto per) {
        return launch_overlapped(route_backward_kernel<decltype(zero), decltype(per)::value>, grid_of(a->T), kRouteThreads, 0,
                                 reinterpret_cast<cudaStream_t>(stream), p);
    }));
    return CSRSPMM_B200_OK;
}

}  // extern "C"

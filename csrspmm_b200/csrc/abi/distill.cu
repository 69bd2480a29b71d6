// extern "C" entry points for distillation from a teacher's entries (declared in include/csrspmm_b200.h).  No counterpart in the
// reference.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../kernels/distill_kernels.cuh"
#include "csrspmm_b200.h"
#include "pdl.h"
#include "plan.h"

using namespace csrspmm_b200;

namespace {

int refuse(const char* what)
{
    set_last_error("distill: %s", what);
    return CSRSPMM_B200_ERR_BAD_ARG;
}

int check(const csrspmm_b200_distill_args* a)
{
    if (a == nullptr || a->struct_size != sizeof(csrspmm_b200_distill_args)) return refuse("args is null or args.struct_size wrong");
    if (a->T < 0 || a->V < 0 || a->ld < a->V) return refuse("negative size, or ld less than V");
    if (a->nnz < 0 || a->nnz > 0x7fffffffLL) return refuse("0 to 2^31 - 1 entries");
    if (a->logit_type < CSRSPMM_B200_F32 || a->logit_type > CSRSPMM_B200_BF16) return refuse("unknown logit_type");
    if (!(a->temperature > 0.0f) || !std::isfinite(a->temperature) || !std::isfinite(1.0f / a->temperature))
        return refuse("temperature has to be positive and finite, its inverse too");
    if (a->V == 0 && a->nnz > 0) return refuse("entries, but no columns");
    if (a->T > 0 && (a->row_ptr == nullptr || (a->V > 0 && a->logits == nullptr) || (a->nnz > 0 && (a->col_idx == nullptr || a->values == nullptr))))
        return refuse("null pointer");
    return CSRSPMM_B200_OK;
}

DistillParams params(const csrspmm_b200_distill_args* a)
{
    DistillParams p = {};
    p.T = a->T, p.V = a->V, p.nnz = (int)a->nnz;
    p.x = a->logits, p.ldx = a->ld;
    p.row_ptr = a->row_ptr, p.col_idx = a->col_idx, p.values = a->values;
    p.temperature = a->temperature, p.inv_t = 1.0f / a->temperature, p.log_probs = a->log_probs != 0;
    return p;
}

template <class F>
cudaError_t for_type(int type, F&& f)
{
    if (type == CSRSPMM_B200_F32) return f(float());
    if (type == CSRSPMM_B200_F16) return f(__half());
    return f(__nv_bfloat16());
}

// Small CTAs for short rows: four warps read 2048 columns of 2 bytes in one go.
constexpr int kFew = 128, kMany = 512;
bool short_rows(const csrspmm_b200_distill_args* a, int parts) { return a->V / parts <= 8192; }

// CTAs of a row: enough that the chip has two per SM, as long as each has a few thousand columns.
int row_parts(const csrspmm_b200_distill_args* a, int most)
{
    int parts = 1;
    while (parts < most && (long long)a->T * parts < 2 * kSms && a->V / (2 * parts) >= 4096) parts *= 2;
    return parts;
}

template <bool GRADIENT>
cudaError_t launch_loss(const csrspmm_b200_distill_args* a, const DistillParams& p, cudaStream_t st)
{
    const int parts = row_parts(a, kDistillMostCtas);
    const unsigned grid = (unsigned)(a->T * (long long)parts);
    return for_type(a->logit_type, [&](auto zero) {
        using T = decltype(zero);
        if (parts > 1) {
            if (short_rows(a, parts)) return launch_clusters(distill_kernel<T, kFew, GRADIENT, true>, grid, parts, kFew, 0, st, p);
            return launch_clusters(distill_kernel<T, kMany, GRADIENT, true>, grid, parts, kMany, 0, st, p);
        }
        if (short_rows(a, 1)) return launch_overlapped(distill_kernel<T, kFew, GRADIENT, false>, grid, kFew, 0, st, p);
        return launch_overlapped(distill_kernel<T, kMany, GRADIENT, false>, grid, kMany, 0, st, p);
    });
}

int finish(cudaError_t e)
{
    if (e == cudaSuccess) return CSRSPMM_B200_OK;
    set_last_error("distill: launch failed: %s", cudaGetErrorString(e));
    return CSRSPMM_B200_ERR_CUDA;
}

}  // namespace

extern "C" {

int csrspmm_b200_distill(const csrspmm_b200_distill_args* a, float* loss, float* stats, csrspmm_b200_stream_t stream)
{
    if (const int bad = check(a)) return bad;
    if (a->T == 0) return CSRSPMM_B200_OK;
    if (loss == nullptr || (reinterpret_cast<uintptr_t>(stats) & 15u) != 0) return refuse("loss is null, or stats not 16-byte aligned");
    DistillParams p = params(a);
    p.loss = loss, p.stats = reinterpret_cast<float4*>(stats);
    return finish(launch_loss<false>(a, p, reinterpret_cast<cudaStream_t>(stream)));
}

int csrspmm_b200_distill_backward(const csrspmm_b200_distill_args* a, const float* stats, const float* weight, int64_t weight_stride, void* dlogits,
                                  int64_t ldd, csrspmm_b200_stream_t stream)
{
    if (const int bad = check(a)) return bad;
    if (ldd < a->V) return refuse("ldd is less than V");
    if (a->T == 0 || a->V == 0) return CSRSPMM_B200_OK;
    if (stats == nullptr || (reinterpret_cast<uintptr_t>(stats) & 15u) != 0 || weight == nullptr || dlogits == nullptr)
        return refuse("null pointer, or stats not 16-byte aligned");
    DistillParams p = params(a);
    p.stats = const_cast<float4*>(reinterpret_cast<const float4*>(stats));
    p.weight = weight, p.weight_stride = weight_stride, p.dx = dlogits, p.ldd = ldd;
    const int parts = (int)std::max<long long>(1, std::min<long long>(a->V / 4096, std::max<long long>(a->V / 32768, 4LL * kSms / a->T)));
    const unsigned grid = (unsigned)(a->T * (long long)parts);
    return finish(for_type(a->logit_type, [&](auto zero) {
        using T = decltype(zero);
        cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
        if (short_rows(a, parts)) return launch_overlapped(distill_backward_kernel<T, kFew>, grid, kFew, 0, st, p, parts);
        return launch_overlapped(distill_backward_kernel<T, kMany>, grid, kMany, 0, st, p, parts);
    }));
}

int csrspmm_b200_distill_grad(const csrspmm_b200_distill_args* a, const float* weight, int64_t weight_stride, float* loss, void* dlogits, int64_t ldd,
                              csrspmm_b200_stream_t stream)
{
    if (const int bad = check(a)) return bad;
    if (ldd < a->V) return refuse("ldd is less than V");
    if (a->T == 0) return CSRSPMM_B200_OK;
    if (loss == nullptr || weight == nullptr || (a->V > 0 && dlogits == nullptr)) return refuse("null pointer");
    DistillParams p = params(a);
    p.loss = loss, p.weight = weight, p.weight_stride = weight_stride, p.dx = dlogits, p.ldd = ldd;
    return finish(launch_loss<true>(a, p, reinterpret_cast<cudaStream_t>(stream)));
}

}  // extern "C"

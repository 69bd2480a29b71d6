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
    if (!std::isnormal(a->temperature * a->temperature)) return refuse("the square of the temperature has to be in fp32");
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

int element_size(int type) { return type == CSRSPMM_B200_F32 ? 4 : 2; }

// Cuts the rows into `parts`, a power of two; returns the CTAs of T rows.
unsigned cut(const csrspmm_b200_distill_args* a, long long parts, DistillParams* p)
{
    for (p->log_parts = 0; 1LL << p->log_parts < parts;) ++p->log_parts;
    p->per = (int)((a->V + parts - 1) / parts + 63) / 64 * 64;
    return (unsigned)(a->T * parts);
}

// Rows that are few are cut further, down to some thousand columns a part, until every SM has two CTAs.
bool too_few(const csrspmm_b200_distill_args* a, long long parts) { return a->T * parts < 2 * kSms && a->V / (2 * parts) >= 2048; }

cudaError_t launch_gradient(const csrspmm_b200_distill_args* a, DistillParams p, cudaStream_t st)
{
    // vectors that a CTA of each shape holds
    constexpr int kSmall = 128 * 2, kMiddle = 128 * 8, kLarge = 256 * 8;
    const int per_vector = 16 / element_size(a->logit_type);
    long long parts = 1;
    while (a->V > parts * kLarge * per_vector || too_few(a, parts)) parts *= 2;  // parts are rounded to 64 columns, which divide kLarge vectors
    const unsigned grid = cut(a, parts, &p);
    const int vectors = p.per / per_vector;
    return for_type(a->logit_type, [&](auto zero) {
        using T = decltype(zero);
        if (vectors <= kSmall) return launch_overlapped(distill_gradient_kernel<T, 128, 2>, grid, 128, 0, st, p);
        if (vectors <= kMiddle) return launch_overlapped(distill_gradient_kernel<T, 128, 8>, grid, 128, 0, st, p);
        return launch_overlapped(distill_gradient_kernel<T, 256, 8>, grid, 256, 0, st, p);
    });
}

constexpr int kPartBytes = 100 * 1024;    // of a part, as far as clusters go: two CTAs of one slot fit an SM (three of up to 64 KB)
constexpr int kFewBytes = 32768;          // up to here four warps do as well as eight, and six CTAs fit an SM (9000 bf16 columns: 192 -> 143 us for 16384 rows)
constexpr int kDynamicSmem = 216 * 1024;  // of a CTA, beside RingShared

// The ring kernel's manager is one warp, and holds up to kListed entries of a row in shared memory; where rows have more, all warps of the long kernel
// walk over them.  Loss and gradient with 256, 384 and 1024 entries a row of bf16 logits, by the ring and by the long kernel: 16384 rows of 3000 columns 261, 531, 1285
// and 304, 328, 471 us, of 9000 282, 747, 1947 and 355, 374, 545, 4096 of 30000 124, 316, 752 and 149, 152, 202, 2048 of 131072 270, 640, 1481
// and 355, 360, 443, 64 of 131072 15, 24, 51 and 19, 20, 25.  With 32 the ring takes 0.4 to 0.65 of the other's time, but for 128 of 600000 (115 and 92).
constexpr int kMostEntries = kListed;
// And where one row may hold so many that its manager's walks over them (four before the workers go on, each up to 20 cycles an entry: 2.7e9 cycles)
// come near the limit of the waits for it, 2^28 attempts of 20 cycles and more.
constexpr long long kMostWalked = 1LL << 25;

template <class T, int WORKERS, bool GRADIENT>
cudaError_t launch_ring(const csrspmm_b200_distill_args* a, DistillParams p, int ctas_per_sm, cudaStream_t st)
{
    constexpr auto kernel = distill_ring_kernel<T, WORKERS, GRADIENT>;
    const int parts = 1 << p.log_parts;
    // A few waves of clusters, so that the SMs end together, of two to four rows each where there are as many.
    p.rows = (int)std::clamp<long long>(((long long)a->T * parts) / ((long long)kSms * ctas_per_sm * 3), 1, WORKERS <= 128 ? kMostRows : 2);
    p.slots = WORKERS <= 128 ? std::min(p.rows, 2) : 1;
    const size_t smem = (size_t)p.ring_offset + (size_t)p.slots * p.slot_bytes;
    const cudaError_t e = allow_dynamic_smem<kernel>(smem);
    if (e != cudaSuccess) return e;
    const unsigned clusters = (unsigned)(((long long)a->T + p.rows - 1) / p.rows);
    return launch_clusters(kernel, clusters * (unsigned)parts, (unsigned)parts, WORKERS + 32, smem, st, p);
}

template <bool GRADIENT>
cudaError_t launch_loss(const csrspmm_b200_distill_args* a, DistillParams p, cudaStream_t st)
{
    const int size = element_size(a->logit_type);
    long long parts = 1;
    while (parts < kDistillMostCtas && ((long long)a->V * size > parts * kPartBytes || too_few(a, parts))) parts *= 2;
    const unsigned grid = cut(a, parts, &p);
    if (parts == 1 && a->V <= 32 * 8 * (16 / size)) {
        const unsigned ctas = (unsigned)(((long long)a->T + kShortThreads / 32 - 1) / (kShortThreads / 32));
        return for_type(a->logit_type, [&](auto zero) {
            using T = decltype(zero);
            if (a->V <= 32 * 2 * (16 / size)) return launch_overlapped(distill_short_kernel<T, 2, GRADIENT>, ctas, kShortThreads, 0, st, p);
            return launch_overlapped(distill_short_kernel<T, 8, GRADIENT>, ctas, kShortThreads, 0, st, p);
        });
    }
    const long long slot = (long long)p.per * size, before = GRADIENT ? ((long long)p.per / 32 + 1 + 31) / 32 * 128 : 0;
    if (before + slot > kDynamicSmem || a->nnz / std::max(a->T, 1) > kMostEntries || a->nnz > kMostWalked)
        return for_type(a->logit_type, [&](auto zero) {
            return launch_clusters(distill_long_kernel<decltype(zero), GRADIENT>, grid, (unsigned)parts, kLongThreads, 0, st, p);
        });
    p.slot_bytes = (int)slot;
    p.ring_offset = (int)before;
    p.wait_limit = wait_limit(kWaitSpinLimit);
    return for_type(a->logit_type, [&](auto zero) {
        using T = decltype(zero);
        if (p.slot_bytes <= kFewBytes) return launch_ring<T, 128, GRADIENT>(a, p, 6, st);
        if (p.slot_bytes <= kPartBytes) return launch_ring<T, 256, GRADIENT>(a, p, p.slot_bytes <= 65536 ? 3 : 2, st);
        return launch_ring<T, 512, GRADIENT>(a, p, 1, st);
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
    return finish(launch_gradient(a, p, reinterpret_cast<cudaStream_t>(stream)));
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

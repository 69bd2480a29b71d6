// extern "C" entry point for the gradient of a product for the matrix's stored values (declared in
// include/csrspmm_b200.h).  No counterpart in the reference.
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "../kernels/sddmm_kernel.cuh"
#include "csrspmm_b200.h"
#include "pdl.h"
#include "plan.h"

using namespace csrspmm_b200;

namespace {

// Where the small product with the transpose is the better way: it must not lose where one column holds all entries either, of which the host knows
// nothing, and its warps must not be more than some waves.  us on the GPU, this kernel and transposition with product (which take 22 from the host,
// this one 8), entries spread evenly and all in one column:
//   2048 entries, 64 columns, 512 of G 8 and 19, 19 and 24; 1000 columns, 64 of G 7 and 17, 20 and 19; 4096 entries in one column 35 to 37 and 21 to 34
//   8192 warps: 1024 entries of 1024 columns, 512 of G 11 and 16, 20 and 22; 2048 of 2048, 64 of G 10 and 15
//   16384 warps: 512 entries of 4096 columns, 512 of G 14 and 19, 21 and 20; 2048 of 1000, 512 of G 19 and 19, 23 and 25; 32768: 32 and 17
constexpr long long kTransposedMostEntries = 2048;
constexpr double kTransposedMostWarps = 1 << 14;

template <int L, int NV, int VW, bool LOOP>
cudaError_t launch(SddmmParams p, cudaStream_t st)
{
    constexpr int groups = kSddmmThreads / L;
    // whole waves of the four CTAs that an SM runs, each with the same number of entries, as many as the row table holds at most
    const long long wave = 4LL * kSms, waves = (p.nnz + wave * kSddmmMostEntries - 1) / (wave * kSddmmMostEntries);
    const long long per_group = std::clamp<long long>((p.nnz + waves * wave * groups - 1) / (waves * wave * groups), 1, kSddmmMostEntries / groups);
    p.run = (int)per_group * groups;
    const unsigned grid = (unsigned)(((long long)p.nnz + p.run - 1) / p.run);
    return launch_overlapped(sddmm_kernel<L, NV, VW, LOOP>, grid, kSddmmThreads, 0, st, p);
}

template <int VW>
cudaError_t launch_width(const SddmmParams& p, cudaStream_t st)
{
    if (p.nvec <= 8) return launch<8, 1, VW, false>(p, st);
    if (p.nvec <= 16) return launch<8, 2, VW, false>(p, st);
    if (p.nvec <= 32) return launch<8, 4, VW, false>(p, st);
    if (p.nvec <= 64) return launch<16, 4, VW, false>(p, st);
    if (p.nvec <= 128) return launch<32, 4, VW, false>(p, st);
    return launch<32, 4, VW, true>(p, st);
}

}  // namespace

extern "C" int csrspmm_b200_sddmm(int32_t M, int32_t Kd, int32_t Nd, int64_t nnz, const int32_t* row_ptr, const int32_t* col_idx, const float* G,
                                  int64_t ldg, const float* B, int64_t ldb, float alpha, float* out, csrspmm_b200_stream_t stream)
{
    if (M < 0 || Kd < 0 || Nd < 0 || nnz < 0 || nnz > 0x7fffffffLL || ldg < Nd || ldb < Nd || (nnz > 0 && (M == 0 || Kd == 0)) ||
        (nnz > 0 && (row_ptr == nullptr || col_idx == nullptr || out == nullptr || (Nd > 0 && (G == nullptr || B == nullptr))))) {
        set_last_error("sddmm: bad argument");
        return CSRSPMM_B200_ERR_BAD_ARG;
    }
    if (nnz == 0) return CSRSPMM_B200_OK;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const auto on = [&](int floats) {
        return Nd % floats == 0 && ldg % floats == 0 && ldb % floats == 0 &&
               ((reinterpret_cast<uintptr_t>(G) | reinterpret_cast<uintptr_t>(B)) & (floats * 4 - 1)) == 0;
    };
    SddmmParams p = {};
    p.M = M, p.Kd = Kd, p.nnz = (int)nnz;
    p.row_ptr = row_ptr, p.col_idx = col_idx;
    p.G = G, p.ldg = ldg, p.B = B, p.ldb = ldb, p.alpha = alpha, p.out = out;
    const int width = on(4) ? 4 : on(2) ? 2 : 1;
    p.nvec = Nd / width;
    const cudaError_t e = width == 4 ? launch_width<4>(p, st) : width == 2 ? launch_width<2>(p, st) : launch_width<1>(p, st);
    if (e != cudaSuccess) {
        set_last_error("sddmm: launch failed: %s", cudaGetErrorString(e));
        return CSRSPMM_B200_ERR_CUDA;
    }
    return CSRSPMM_B200_OK;
}

// What the warps of the small product with the transpose divide: groups of rows of C times parts of 32 vectors of `width` floats ...
static long long transposed_parts(int32_t Kd, int32_t Nd, int width)
{
    return ((long long)Kd + kTransposedRows - 1) / kTransposedRows * (((long long)Nd / width + 31) / 32);
}
// ... each in as many runs of the entries, as a power of two.
static int log_pieces(int64_t nnz)
{
    int n = 0;
    while (1 << n < kTransposedThreads / 32 && (int64_t)kTransposedRun << n < nnz) ++n;
    return n;
}

extern "C" int csrspmm_b200_spmm_transposed_pays(int32_t Kd, int32_t Nd, int64_t nnz)
{
    if (Kd < 0 || Nd < 0 || nnz < 0 || nnz > kTransposedMostEntries) return 0;
    return (double)transposed_parts(Kd, Nd, Nd % 4 == 0 ? 4 : Nd % 2 == 0 ? 2 : 1) * (1 << log_pieces(nnz)) <= kTransposedMostWarps;
}

extern "C" int csrspmm_b200_spmm_transposed(int32_t M, int32_t Kd, int32_t Nd, int64_t nnz, const int32_t* row_ptr, const int32_t* col_idx,
                                            const float* values, const float* G, int64_t ldg, float alpha, float* C, int64_t ldc,
                                            csrspmm_b200_stream_t stream)
{
    if (M < 0 || Kd < 0 || Nd < 0 || nnz < 0 || nnz > 0x7fffffffLL || ldg < Nd || ldc < Nd || (nnz > 0 && (M == 0 || Kd == 0)) ||
        (Kd > 0 && Nd > 0 && (C == nullptr || (nnz > 0 && (row_ptr == nullptr || col_idx == nullptr || values == nullptr || G == nullptr))))) {
        set_last_error("spmm_transposed: bad argument");
        return CSRSPMM_B200_ERR_BAD_ARG;
    }
    if (Kd == 0 || Nd == 0) return CSRSPMM_B200_OK;
    const auto on = [&](int floats) {
        return Nd % floats == 0 && ldg % floats == 0 && ldc % floats == 0 &&
               ((reinterpret_cast<uintptr_t>(G) | reinterpret_cast<uintptr_t>(C)) & (floats * 4 - 1)) == 0;
    };
    const int width = on(4) ? 4 : on(2) ? 2 : 1;
    const int pieces = log_pieces(nnz), per_cta = (kTransposedThreads / 32) >> pieces;
    const int run = (int)((nnz + (32LL << pieces) - 1) / (32LL << pieces)) * 32;
    const TransposedParams p = {M, Kd, Nd / width, (int)nnz, row_ptr, col_idx, values, G, ldg, alpha, C, ldc, pieces, run};
    const long long ctas = (transposed_parts(Kd, Nd, width) + per_cta - 1) / per_cta;
    if (ctas > 0x7fffffffLL) {
        set_last_error("spmm_transposed: too many rows and columns");
        return CSRSPMM_B200_ERR_UNSUPPORTED;
    }
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const cudaError_t e = width == 4   ? launch_overlapped(spmm_transposed_kernel<4>, (unsigned)ctas, kTransposedThreads, 0, st, p)
                          : width == 2 ? launch_overlapped(spmm_transposed_kernel<2>, (unsigned)ctas, kTransposedThreads, 0, st, p)
                                       : launch_overlapped(spmm_transposed_kernel<1>, (unsigned)ctas, kTransposedThreads, 0, st, p);
    if (e != cudaSuccess) {
        set_last_error("spmm_transposed: launch failed: %s", cudaGetErrorString(e));
        return CSRSPMM_B200_ERR_CUDA;
    }
    return CSRSPMM_B200_OK;
}

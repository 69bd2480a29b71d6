// The 64-bit exponential and reciprocal of the routing kernel (csrc/kernels/route_kernels.cuh) against long double, over all that they are given:
// arguments from 0 to far below the smallest number, and sums of 1 to 1024 scores.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "../../csrspmm_b200/csrc/kernels/route_kernels.cuh"

__global__ void exponentials(const double* in, double* out, int n)
{
    const int i = (int)(blockIdx.x * blockDim.x + threadIdx.x);
    if (i < n) out[i] = csrspmm_b200::exp_of_negative(in[i]);
}

__global__ void reciprocals(const double* in, double* out, int n)
{
    const int i = (int)(blockIdx.x * blockDim.x + threadIdx.x);
    if (i < n) out[i] = csrspmm_b200::reciprocal(in[i]);
}

// The largest difference in units of the last place of the result (of the smallest number, where the result is below the normal ones)
template <class Want>
static double worst(void (*kernel)(const double*, double*, int), const std::vector<double>& in, Want&& want)
{
    const int n = (int)in.size();
    double *x = nullptr, *y = nullptr;
    if (cudaMalloc(&x, n * sizeof(double)) != cudaSuccess || cudaMalloc(&y, n * sizeof(double)) != cudaSuccess) return HUGE_VAL;
    std::vector<double> got(n);
    cudaMemcpy(x, in.data(), n * sizeof(double), cudaMemcpyHostToDevice);
    kernel<<<(n + 255) / 256, 256>>>(x, y, n);
    const cudaError_t e = cudaMemcpy(got.data(), y, n * sizeof(double), cudaMemcpyDeviceToHost);
    cudaFree(x);
    cudaFree(y);
    if (e != cudaSuccess) return HUGE_VAL;
    double most = 0.0;
    for (int i = 0; i < n; ++i) {
        const long double w = want((long double)in[i]);
        int exponent;
        frexpl(w, &exponent);  // w = f 2^exponent, 0.5 <= f < 1: its unit is 2^(exponent - 53), or 2^-1074
        const int unit = w == 0.0L || exponent - 53 < -1074 ? -1074 : exponent - 53;
        const double off = (double)fabsl(ldexpl((long double)got[i] - w, -unit));
        if (!(off <= most)) most = std::isnan(off) ? HUGE_VAL : off;
    }
    return most;
}

int main()
{
    std::mt19937_64 rng(1);
    std::vector<double> x = {0.0, -0.0, -1e-300, -1e-17, -0.34657359027997264, -0.34657359027997270, -708.0, -709.5, -745.0, -745.2, -746.0, -1399.9, -1400.0, -1e4, -3e38};
    for (const double least : {1e-12, 1e-3, 1.0, 40.0, 708.0, 760.0, 1500.0})
        for (int i = 0; i < 100000; ++i) x.push_back(-least * std::uniform_real_distribution<double>(0.0, 1.0)(rng));
    for (int n = 0; n < 2100; ++n)  // next to the borders of the reduction
        for (const double d : {-1e-13, 0.0, 1e-13}) x.push_back(-(n + 0.5) * 0.6931471805599453 - d);
    std::vector<double> v = {1.0, 1.0 + 0x1p-52, 2.0, 3.0, 1023.0, 1024.0, 1048575.0};
    for (int i = 0; i < 300000; ++i) v.push_back(std::exp2(std::uniform_real_distribution<double>(0.0, 20.0)(rng)));
    const double e = worst(exponentials, x, [](long double a) { return expl(a); }), r = worst(reciprocals, v, [](long double a) { return 1.0L / a; });
    std::printf("exponential %.3f units, reciprocal %.3f units\n", e, r);
    // exponential: half a unit for the last step of the series, at most as much for those before it, whose sum is r or less, 0.35 of two halves for r, and where the
    // unit is the smallest number half of one for the second factor; a unit is at most twice as much relative to the result.  Reciprocal: half a unit for the last
    // step and 2^-40 of a unit for what Newton's step leaves of the one before.
    return e <= 2.0 && r <= 1.5 ? 0 : 1;
}

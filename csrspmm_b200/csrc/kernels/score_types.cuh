// What the kernels on dense rows of scores share (routing, distillation): the element types, 16-byte vectors of
// them, reductions of a warp.  Everything is computed in fp32; a result is rounded to its type once.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace csrspmm_b200 {

constexpr unsigned kAllLanes = 0xffffffffu;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v)
{
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}

// N elements that are read and written at once, at a multiple of their size
template <class T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

// 16 bytes of a row, read once and kept out of L1
__device__ __forceinline__ uint4 load_once(const void* p)
{
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Two fp32 numbers that are computed with at once
struct Pair {
    unsigned long long v;
};
__device__ __forceinline__ Pair pair_of(float a, float b)
{
    Pair r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 halves(Pair a)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c)
{
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b)
{
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b)
{
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}

// 16 bytes of a row: four fp32 elements, or eight 16-bit ones, the lower half of a word first.
template <class T>
struct Words;
template <>
struct Words<float> {
    static constexpr unsigned kMinusInf = 0xff800000u, kNaN = 0x7fffffffu;
    static __device__ __forceinline__ unsigned max(unsigned a, unsigned b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ float largest(unsigned a) { return __uint_as_float(a); }
    template <class F>
    static __device__ __forceinline__ void each(const uint4& a, F&& f)
    {
        f(pair_of(__uint_as_float(a.x), __uint_as_float(a.y)));
        f(pair_of(__uint_as_float(a.z), __uint_as_float(a.w)));
    }
    template <class F>
    static __device__ __forceinline__ uint4 map(const uint4& a, F&& f)
    {
        const float2 u = halves(f(pair_of(__uint_as_float(a.x), __uint_as_float(a.y)))), v = halves(f(pair_of(__uint_as_float(a.z), __uint_as_float(a.w))));
        return make_uint4(__float_as_uint(u.x), __float_as_uint(u.y), __float_as_uint(v.x), __float_as_uint(v.y));
    }
};

template <class T, class T2>
struct HalfWords {
    static __device__ __forceinline__ T2 both(unsigned a) { return *reinterpret_cast<T2*>(&a); }
    static __device__ __forceinline__ unsigned max(unsigned a, unsigned b)  // of a number and a NaN the number
    {
        const T2 r = __hmax2(both(a), both(b));
        return *reinterpret_cast<const unsigned*>(&r);
    }
    static __device__ __forceinline__ Pair wide(unsigned a)
    {
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            return pair_of(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u));
        } else {
            const float2 v = __half22float2(both(a));
            return pair_of(v.x, v.y);
        }
    }
    static __device__ __forceinline__ unsigned narrow(Pair a)
    {
        const float2 v = halves(a);
        T2 r;
        if constexpr (std::is_same_v<T, __nv_bfloat16>) r = __floats2bfloat162_rn(v.x, v.y);
        else r = __floats2half2_rn(v.x, v.y);
        return *reinterpret_cast<const unsigned*>(&r);
    }
    static __device__ __forceinline__ float largest(unsigned a)
    {
        const float2 v = halves(wide(a));
        return fmaxf(v.x, v.y);
    }
    template <class F>
    static __device__ __forceinline__ void each(const uint4& a, F&& f)
    {
        f(wide(a.x));
        f(wide(a.y));
        f(wide(a.z));
        f(wide(a.w));
    }
    template <class F>
    static __device__ __forceinline__ uint4 map(const uint4& a, F&& f)
    {
        return make_uint4(narrow(f(wide(a.x))), narrow(f(wide(a.y))), narrow(f(wide(a.z))), narrow(f(wide(a.w))));
    }
};
template <>
struct Words<__nv_bfloat16> : HalfWords<__nv_bfloat16, __nv_bfloat162> {
    static constexpr unsigned kMinusInf = 0xff80ff80u, kNaN = 0x7fff7fffu;
};
template <>
struct Words<__half> : HalfWords<__half, __half2> {
    static constexpr unsigned kMinusInf = 0xfc00fc00u, kNaN = 0x7fff7fffu;
};

// The largest of 16 bytes' elements and `top`, by words
template <class T>
__device__ __forceinline__ unsigned max_words(unsigned top, const uint4& v)
{
    return Words<T>::max(Words<T>::max(top, Words<T>::max(v.x, v.y)), Words<T>::max(v.z, v.w));
}

// of numbers and NaNs the largest number
__device__ __forceinline__ float warp_max(float v)
{
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

template <class F>
__device__ __forceinline__ F warp_sum(F v)
{
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kAllLanes, v, d);
    return v;
}

}  // namespace csrspmm_b200

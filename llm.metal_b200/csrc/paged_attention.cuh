// What the kernels of attention over pages share: elements of the cache's type.
#pragma once
#include "paged_plan.cuh"

#include <cuda_bf16.h>

#include <limits.h>
#include <type_traits>

namespace {

__device__ __forceinline__ float ex2(float x)                // 2^x, 2 ulp, 0 for -inf
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
template <typename T> __device__ __forceinline__ float to_float(uint16_t b)
{
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half(b));
    else return __uint_as_float((uint32_t)b << 16);
}
// Weights are powers of two over the largest score so far, less this: binary16 ends at 2^15.99 above and has its full precision down to 2^-14 only, so that of weights of 1 at most half
// its range would lie idle, and 65 536 keys of 2^-26 each, 2^-10 of the sum together, would vanish from the weighted one. `most`: such that the largest weight is 2^15. bfloat16 has fp32's range.
template <typename T> __device__ __forceinline__ constexpr float weight_lift(int most) { return std::is_same<T, __half>::value ? (float)most : 0.0f; }
// Whether one of the eight elements of a 16-byte word is infinite or NaN.
template <typename T> __device__ __forceinline__ bool any_special(const uint4 &v)
{
    constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= (w[i] & E) == E || ((w[i] >> 16) & E) == E;
    return any;
}

}  // namespace

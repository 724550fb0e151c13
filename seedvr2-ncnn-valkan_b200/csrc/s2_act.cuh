// Element types and activations shared by the channels-last operators
// (s2_group_norm.cu, s2_linear.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "s2_b200.h"

namespace s2dev {

// fp32 values of a 16-bit or 32-bit element, and one rounding (to nearest even) back.
template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ float to_float<__half>(__half v)
{
    return __half2float(v);
}
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v)
{
    return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v)
{
    return v;
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v)
{
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v)
{
    return __float2bfloat16_rn(v);
}

// Two 16-bit values of a 32-bit word <-> two floats (element 0 in the low half).
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t u)
{
    return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u)
{
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// The activations in fp32. silu and gelu_tanh divide by 1 + e^-z, with the hardware's
// exponential and division (a few 2^-23 relative each, far below an output's rounding to
// 16 bits); a negative argument whose e^-z overflows gives -0, as the formula does.
// A NaN stays a NaN, under relu too.
template <int kAct>
__device__ __forceinline__ float activate(float v)
{
    if constexpr (kAct == S2_ACT_RELU) return v < 0.f ? 0.f : v;
    if constexpr (kAct == S2_ACT_SILU) return __fdividef(v, 1.f + __expf(-v));
    if constexpr (kAct == S2_ACT_GELU) {
        // erfc(u) = t (a1 + t (a2 + ... + t a5)) e^-u^2, t = 1 / (1 + 0.3275911 u), u >= 0, within
        // 1.5e-7 (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26); here u = |v| /
        // sqrt 2, and 1 + erf(v / sqrt 2) is erfc(u) below 0 and 2 - erfc(u) above: nothing cancels.
        // A third of erff's instructions, one branch-free run: the product at 21600 x 10240 x 2560
        // spends 4500 of a tile's 20500 cycles on its activation with erff.
        const float t = __fdividef(1.f, fmaf(0.3275911f * 0.70710678118654752f, fabsf(v), 1.f));
        float p = fmaf(t, 1.061405429f, -1.453152027f);
        p = fmaf(t, p, 1.421413741f);
        p = fmaf(t, p, -0.284496736f);
        p = fmaf(t, p, 0.254829592f);
        const float c = p * t * __expf(-0.5f * v * v);
        return 0.5f * v * (v >= 0.f ? 2.f - c : c);
    }
    if constexpr (kAct == S2_ACT_GELU_TANH) {
        // 0.5 v (1 + tanh u) = v / (1 + e^-2u), u = sqrt(2 / pi) (v + 0.044715 v^3)
        const float u2 = 1.5957691216057308f * v * (1.f + 0.044715f * v * v);
        return __fdividef(v, 1.f + __expf(-u2));
    }
    return v;
}

}  // namespace s2dev

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

// Two floats in one 64-bit register: one instruction works on both.
__device__ __forceinline__ uint64_t pair(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 floats_of(uint64_t p)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t both(float a) { return pair(a, a); }

// 2^x and 1 / x as the hardware gives them (2^-22 relative). The .ftz forms: without it each takes four
// more instructions for denormals, which change nothing here (2^x of a denormal is 1).
__device__ __forceinline__ uint64_t ex2_2(uint64_t x)
{
    float2 f = floats_of(x);
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(f.x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(f.y));
    return pair(f.x, f.y);
}
__device__ __forceinline__ uint64_t rcp_2(uint64_t x)
{
    float2 f = floats_of(x);
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(f.x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(f.y));
    return pair(f.x, f.y);
}

// The activations of two values in fp32. Relative errors, in units of 2^-23: relu 0; silu 6 + |v|; gelu
// 8 + v^2 / 2; gelu_tanh 6 + 2 w, w = 2 sqrt(2 / pi) (|v| + 0.044715 |v|^3); above 0 two more and not the second
// terms, which come from rounding the exponents of e^-v, e^(-v^2 / 2) and e^w, as a rounding of v itself would. Results below 2^-119 may come out as 0 of their sign (-0 where e^-v overflows, as in the formulas). A
// NaN stays a NaN, under relu too.
template <int kAct>
__device__ __forceinline__ uint64_t activate2(uint64_t v)
{
    constexpr float kLog2e = 1.4426950408889634f;
    if constexpr (kAct == S2_ACT_RELU) {
        const float2 f = floats_of(v);
        return pair(f.x < 0.f ? 0.f : f.x, f.y < 0.f ? 0.f : f.y);
    }
    if constexpr (kAct == S2_ACT_SILU)  // v / (1 + e^-v)
        return mul2(v, rcp_2(add2(ex2_2(mul2(v, both(-kLog2e))), both(1.f))));
    if constexpr (kAct == S2_ACT_GELU_TANH) {
        // 0.5 v (1 + tanh u) = v / (1 + e^-2u), u = sqrt(2 / pi) (v + 0.044715 v^3)
        const uint64_t u = mul2(v, fma2(mul2(v, v), both(-2.f * 0.7978845608028654f * 0.044715f * kLog2e),
                                        both(-2.f * 0.7978845608028654f * kLog2e)));
        return mul2(v, rcp_2(add2(ex2_2(u), both(1.f))));
    }
    if constexpr (kAct == S2_ACT_GELU) {
        // h = erfc(|v| / sqrt 2) / 2 = e^(-v^2 / 2) t P(t), t = 1 / (1 + 0.305 |v|): gelu is v h below 0 and
        // v (1 - h) above, so nothing cancels. P is our own minimax fit (degree 7, relative error 9.4e-8) over the
        // |v| <= 13.25 whose e^(-v^2 / 2) is a normal fp32 value; past them h is 0.
        const float2 f = floats_of(v);
        const uint64_t t = rcp_2(fma2(pair(fabsf(f.x), fabsf(f.y)), both(0.305f), both(1.f)));
        uint64_t p = fma2(t, both(0.03669919239924065f), both(-0.152988317866804f));
        p = fma2(t, p, both(0.18571690732108168f));
        p = fma2(t, p, both(-0.03797682777863402f));
        p = fma2(t, p, both(0.1210216757736468f));
        p = fma2(t, p, both(0.10342086782285753f));
        p = fma2(t, p, both(0.12246681664173774f));
        p = fma2(t, p, both(0.1216397326792894f));
        const uint64_t h = mul2(mul2(p, t), ex2_2(mul2(mul2(v, v), both(-0.5f * kLog2e))));
        const float2 lo = floats_of(h), hi = floats_of(fma2(h, both(-1.f), both(1.f)));
        return mul2(v, pair(f.x >= 0.f ? hi.x : lo.x, f.y >= 0.f ? hi.y : lo.y));
    }
    return v;
}
template <int kAct>
__device__ __forceinline__ float activate(float v)
{
    return floats_of(activate2<kAct>(pair(v, v))).x;
}

}  // namespace s2dev

// abh_choice.hpp -- what the kernels share that choose a token's largest logits: their order, and the softmax's exponential.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "abh_device.hpp"
#include "abh_rows.hpp"

namespace abh {

constexpr float kRouteLog2e = 1.4426950408889634f;
constexpr float kRouteNegInf = -__builtin_inff();

// A total order of floats as integers: -inf lowest but 0 (nothing), +0 and -0 equal, NaN above all.
__device__ __forceinline__ uint32_t order_key(float x)
{
    if (x != x) return 0xffffffffu;
    const uint32_t u = fbits(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float key_value(uint32_t key)
{
    return key == 0xffffffffu ? __builtin_nanf("") : bitsf(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// exp(x - m) with m = -inf taken as 0, so that a row without any finite logit has weights 0 and not NaN.  x - m and its
// product with log2 e are rounded to FP32: the largest weight's exponential is exact, one of e^-8 is off by at most 2^-20 of
// itself, one near FP32's smallest, e^-87, by 2^-17.
__device__ __forceinline__ float exp_below(float x, float m)
{
    return __builtin_amdgcn_exp2f((x - (m == kRouteNegInf ? 0.0f : m)) * kRouteLog2e);
}

template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t x)
{
    return group_reduce<G>(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

}  // namespace abh

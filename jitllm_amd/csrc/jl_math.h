// Functions that more than one kernel evaluates.
#pragma once

#include "jl_device.h"

// The series of tanh, odd powers up to the 13th, where |x| <= kTanhNear (its next term is below 2^-25 of the value), else
// (1 - e) / (1 + e), e = exp(-2 |x|), in whose difference nothing much cancels by then: each within 2^-21 of the value.
constexpr float kTanhNear = 0.4f;
__device__ __forceinline__ float jl_tanh_near(float x) {
    const float y = x * x;
    float near = fmaf(y, 21844.f / 6081075.f, -1382.f / 155925.f);
    near = fmaf(y, near, 62.f / 2835.f);
    near = fmaf(y, near, -17.f / 315.f);
    near = fmaf(y, near, 2.f / 15.f);
    near = fmaf(y, near, -1.f / 3.f);
    return fmaf(x * y, near, x);
}
__device__ __forceinline__ float jl_tanh(float x) {
    const float e = __builtin_amdgcn_exp2f(-2.88539008177792681472f * fabsf(x));
    const float far = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), x);
    return fabsf(x) <= kTanhNear ? jl_tanh_near(x) : far;
}

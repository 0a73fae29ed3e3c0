// Functions that more than one kernel evaluates.
#pragma once

#include "jl_device.h"

// tanh.  Up to kTanhMiddle, Lambert's continued fraction x / (1 + y / (3 + y / (5 + ... y / 13))), y = x^2, as one quotient:
// off by 1.3e-7 of the value there, and far less below.  Beyond, (1 - e) / (1 + e) with e = exp(-2 |x|), in whose
// difference nothing much cancels from 1 on.  Each is within 2^-21 of the value.
constexpr float kTanhMiddle = 2.5f;
__device__ __forceinline__ float jl_tanh_middle(float x) {
    const float y = x * x;
    const float over = fmaf(y, fmaf(y, y + 378.f, 17325.f), 135135.f);
    const float under = fmaf(y, fmaf(y, fmaf(y, 28.f, 3150.f), 62370.f), 135135.f);
    return x * over * __builtin_amdgcn_rcpf(under);
}
__device__ __forceinline__ float jl_tanh(float x) {
    const float e = __builtin_amdgcn_exp2f(-2.88539008177792681472f * fabsf(x));
    const float far = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), x);
    return fabsf(x) <= 1.f ? jl_tanh_middle(x) : far;
}

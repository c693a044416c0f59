// exl3_activation.hpp -- device exponentials, sigmoids and inverse roots in binary32.
#pragma once

#include "exl3_device.hpp"

namespace exl3k {

// exp(x) to about 2 ulp: v_exp_f32 of the rounded x log2(e), times 1 + ln(2) times that product's
// error (v_exp_f32 of the product alone is off by 2^-24 of the exponent: 8e-7 at x = 10).  Beyond
// |x| = 200 the result is the limit's, 0 or infinity; NaN counts as -200.
__device__ __forceinline__ float exp_f32(float x) {
    constexpr double l = 1.44269504088896340736;
    constexpr float hi = (float)l, lo = (float)(l - (double)hi);
    x = fminf(fmaxf(x, -200.f), 200.f);
    const float p = x * hi;
    const float e = __builtin_fmaf(x, lo, __builtin_fmaf(x, hi, -p));
    return __builtin_amdgcn_exp2f(p) * __builtin_fmaf(e, 0.693147180559945f, 1.f);
}

// 1 / (1 + exp(-z)); a NaN stays one in silu by its factor
__device__ __forceinline__ float sigmoid_f32(float z) { return __builtin_amdgcn_rcpf(1.f + exp_f32(-z)); }
__device__ __forceinline__ float silu_f32(float z) { return z * sigmoid_f32(z); }

// 1 / sqrt(x): v_rsq_f32 is good to 1 ulp, of normal numbers
__device__ __forceinline__ float inverse_root(float x) {
    const bool tiny = x < 0x1p-100f;
    return __builtin_amdgcn_rsqf(tiny ? x * 0x1p64f : x) * (tiny ? 0x1p32f : 1.f);
}

}  // namespace exl3k

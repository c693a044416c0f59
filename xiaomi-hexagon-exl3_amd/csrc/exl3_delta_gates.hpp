// exl3_delta_gates.hpp -- device helpers of the delta rule's kernels: gates and inverse lengths.
#pragma once

#include <math.h>

#include "exl3_activation.hpp"
#include "exl3_packed_rows.hpp"

namespace exl3k {

// log(1 + exp(x))
__device__ __forceinline__ float softplus_f32(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

// A row's log decay and beta for one head.  From -200 down the decay is 0 in binary32, and sums of
// such logs stay finite; a NaN stays one.
struct Gates {
    float g, beta;
};
__device__ __forceinline__ Gates gates_of(const DeltaArgs &a, size_t row, int head) {
    const size_t at = row * a.gate_stride + head;
    float g = a.g[at], beta = a.beta[at];
    if (a.a_log) {
        const float x = g + a.dt_bias[head];
        g = x == x ? -expf(a.a_log[head]) * softplus_f32(x) : x;
        beta = 1.f / (1.f + expf(-beta));
    }
    return {g < -200.f ? -200.f : g, beta};
}
// exp of a log decay (or a sum of them); NaN stays one
__device__ __forceinline__ float decay_of(float g) { return g == g ? exp_f32(g) : g; }

// 1 / sqrt(sum of squares + eps), to 1 ulp
__device__ __forceinline__ float inverse_length(float squares, float eps) {
    const float s = squares + eps;
    const bool tiny = s < 0x1p-100f;
    return __builtin_amdgcn_rsqf(tiny ? s * 0x1p64f : s) * (tiny ? 0x1p32f : 1.f);
}

}  // namespace exl3k

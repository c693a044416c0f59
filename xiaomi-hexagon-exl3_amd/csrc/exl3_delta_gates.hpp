// exl3_delta_gates.hpp -- device helpers of the delta rule's kernels: gates.
#pragma once

#include <math.h>

#include "exl3_activation.hpp"
#include "exl3_packed_rows.hpp"

namespace exl3k {

// log(1 + exp(x))
__device__ __forceinline__ float softplus_f32(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

// A head's part of raw gates, and a row's log decay and beta for it.  From -200 down the decay is 0 in binary32,
// and sums of such logs stay finite; a NaN stays one.
struct HeadGates {
    float rate, bias;
};
__device__ __forceinline__ HeadGates head_gates(const DeltaArgs &a, int head) {
    return a.a_log ? HeadGates{-expf(a.a_log[head]), a.dt_bias[head]} : HeadGates{0.f, 0.f};
}
struct Gates {
    float g, beta;
};
__device__ __forceinline__ Gates load_gates(const DeltaArgs &a, size_t row, int head) {
    const size_t at = row * a.gate_stride + head;
    return {a.g[at], a.beta[at]};
}
__device__ __forceinline__ Gates gates_of(const DeltaArgs &a, const HeadGates &h, Gates r) {
    if (a.a_log) {
        const float x = r.g + h.bias;
        r.g = x == x ? h.rate * softplus_f32(x) : x;
        r.beta = 1.f / (1.f + expf(-r.beta));
    }
    r.g = r.g < -200.f ? -200.f : r.g;
    return r;
}
// exp of a log decay (or a sum of them); NaN stays one
__device__ __forceinline__ float decay_of(float g) { return g == g ? exp_f32(g) : g; }

}  // namespace exl3k

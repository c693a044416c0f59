// exl3_attention_rows.hpp -- attention of one query row by one wave: 64 keys at a time, a key
// per lane, the running maximum and sum of the softmax, then a share of the row per lane.
#pragma once

#include "exl3_head_rows.hpp"

namespace exl3k {

// o[i]: the weighted sum of element 64 i + lane; returns the factor that normalises it (0 for
// a row that sees no key).  `rotate`: the query goes through the cache's H32 first.
template <int D, typename Rows>
__device__ __forceinline__ float attend_row(const _Float16 *q, int rotate, const Rows &rows, int seen, float scale,
                                            float (&o)[D / 64]) {
    __shared__ float qs[D];
    __shared__ float ps[64];
    const int lane = threadIdx.x;
    if (8 * lane < D) {
        float x[8];
        load_run8<1>(q, 8 * lane, 0, x);
        if (rotate) h32_run8(x, lane);
        for (int e = 0; e < 8; ++e) qs[8 * lane + e] = x[e];
    }
    __syncthreads();
    float top = -INFINITY, sum = 0.f;
    for (int i = 0; i < D / 64; ++i) o[i] = 0.f;
    for (int n0 = 0; n0 < seen; n0 += 64) {
        const int n = n0 + lane;
        float s = -INFINITY;
        if (n < seen) {
            float acc = 0.f;
            for (int i = 0; i < D; ++i) acc += qs[i] * rows.key(n, i);
            s = acc * scale;
        }
        const float m = fmaxf(top, wave_max(s));
        const float base = m == -INFINITY ? 0.f : m;
        const float p = n < seen ? __expf(s - base) : 0.f, keep = __expf(top - base);
        float all = p;
        for (int d = 1; d < 64; d <<= 1) all += __shfl_xor(all, d);
        sum = sum * keep + all;
        top = m;
        ps[lane] = p;
        __syncthreads();
        const int count = seen - n0 < 64 ? seen - n0 : 64;
        for (int i = 0; i < D / 64; ++i) {
            float acc = o[i] * keep;
            for (int j = 0; j < count; ++j) acc += ps[j] * rows.value(n0 + j, i * 64 + lane);
            o[i] = acc;
        }
        __syncthreads();
    }
    return seen > 0 ? 1.0f / sum : 0.f;
}

}  // namespace exl3k

// exl3_head_rows.hpp -- device helpers of the attention block's kernels: eight
// consecutive elements of a head per lane, and the H32 rotation of the cache.
#pragma once

#include "exl3_attention.hpp"
#include "exl3_kernel_common.hpp"

namespace exl3k {

// Workgroups for `rows` lane groups, `per` in each: the kernels step through what is beyond
// this grid (a grid has fewer than 2^32 work-items).
inline unsigned row_blocks(size_t rows, size_t per) {
    const size_t blocks = (rows + per - 1) / per, most = (size_t)1 << 22;
    return (unsigned)(blocks < most ? blocks : most);
}

// Elements 8 l .. 8 l + 7 of a head's row, widened to binary32.
template <int F16>
__device__ __forceinline__ void load_run8(const void *p, size_t at, int vec, float (&v)[8]) {
    if constexpr (F16) {
        const _Float16 *h = (const _Float16 *)p + at;
        if (vec) {
            const h8 t = *(const h8 *)h;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (float)t[e];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (float)h[e];
        }
    } else {
        const float *f = (const float *)p + at;
        if (vec) {
            const f4 a = ((const f4 *)f)[0], b = ((const f4 *)f)[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = a[e];
                v[4 + e] = b[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = f[e];
        }
    }
}
template <int F16>
__device__ __forceinline__ void store_run8(void *p, size_t at, int vec, const float (&v)[8]) {
    if constexpr (F16) {
        _Float16 *h = (_Float16 *)p + at;
        h8 t;
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = (_Float16)v[e];
        if (vec) {
            *(h8 *)h = t;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = t[e];
        }
    } else {
        float *f = (float *)p + at;
        if (vec) {
            ((f4 *)f)[0] = (f4){v[0], v[1], v[2], v[3]};
            ((f4 *)f)[1] = (f4){v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = v[e];
        }
    }
}

// H32 of a group of 32 elements held by four lanes (l % 4 = 0 .. 3) of eight: butterflies
// (a + b, a - b) between elements 1, 2, 4 (in the lane), 8 and 16 (lanes l ^ 1 and l ^ 2)
// apart, in this order, then 1/sqrt(32).  The order fixes the bits of every quantised code.
__device__ __forceinline__ void h32_run8(float (&v)[8], int lane) {
#pragma unroll
    for (int step = 1; step < 8; step <<= 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i & step) continue;
            const float a = v[i], b = v[i + step];
            v[i] = a + b;
            v[i + step] = a - b;
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = lane_butterfly<1>(v[i], lane);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = lane_butterfly<2>(v[i], lane) * 0.17677669529663687f;
}

}  // namespace exl3k

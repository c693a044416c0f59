// exl3_head_rows.hpp -- device helpers of the attention block's kernels: eight
// consecutive elements of a head per lane, and the H32 rotation of the cache.
#pragma once

#include "exl3_attention.hpp"
#include "exl3_kernel_common.hpp"

namespace exl3k {

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
// apart, in this order, then 1/sqrt(32).  The order fixes the bits of every quantised code.  The
// two stages between lanes keep the sign of the upper lane for the last product (dpp_block_stage8).
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
    const float s1 = (lane & 1) ? -1.f : 1.f, s2 = (lane & 2) ? -1.f : 1.f;
    dpp_block_stage8<1>(v, s1);
    dpp_block_stage8<2>(v, s2);
    const float scale = s1 * s2 * 0.17677669529663687f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= scale;
}

// Workgroups for `rows` lane groups, `per` in each: the kernels step through what is beyond
// this grid (a grid has fewer than 2^32 work-items).
inline unsigned row_blocks(size_t rows, size_t per) {
    const size_t blocks = (rows + per - 1) / per, most = (size_t)1 << 22;
    return (unsigned)(blocks < most ? blocks : most);
}

// Lane groups take one token each, neighbouring groups neighbouring tokens, and walk
// the rows (heads of q and k, or of keys and values) slice, slice + slices, ..: a workgroup's share of
// `rows` so that `groups` workgroups' worth of lane groups are busy where the rows allow it.  A grid
// has fewer than 2^32 work-items: beyond that the kernels step through the tokens.
struct RowGrid {
    unsigned blocks;
    int slices;
};
inline RowGrid row_grid(size_t tokens, size_t tokens_per_block, size_t rows, size_t groups) {
    const size_t tb = (tokens + tokens_per_block - 1) / tokens_per_block;
    size_t slices = (groups + tb - 1) / tb;
    slices = slices < rows ? slices : rows;
    const size_t blocks = tb * slices, most = ((size_t)1 << 22) / slices * slices;
    return {(unsigned)(blocks < most ? blocks : most), (int)slices};
}

}  // namespace exl3k

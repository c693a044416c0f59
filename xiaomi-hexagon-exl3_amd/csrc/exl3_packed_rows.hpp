// exl3_packed_rows.hpp -- device helpers of the kernels that walk packed sequences in tiles of rows.
#pragma once

#include "exl3_kernel_common.hpp"
#include "exl3_linear_attention.hpp"

namespace exl3k {

// The rows of sequence s, first and count.  starts that are not ascending or not within the
// rows make it empty.
struct Rows {
    int first, count;
};
__device__ __forceinline__ int within(int v, int top) { return v < 0 ? 0 : (v > top ? top : v); }
__device__ __forceinline__ Rows rows_of(const Sequences &p, int s) {
    if (!p.starts) {
        const int n = p.tokens / p.sequences;
        return {s * n, n};
    }
    const int a = within(p.starts[s], p.tokens), b = within(p.starts[s + 1], p.tokens);
    return {a, b > a ? b - a : 0};
}

// Tile t, where each sequence in turn has its rows in tiles of `per`, and one tile where it has no rows:
// the sequence (-1: there is no such tile), its rows and the tile's first row among them.  The wave's lanes ask together.
struct Tile {
    int s, row0;
    Rows rows;
};
__device__ __forceinline__ Tile find_tile(const Sequences &p, int t, int per, int lane) {
    if (!p.starts) {
        const int n = p.tokens / p.sequences, tiles = n > per ? (n + per - 1) / per : 1, s = t / tiles;
        return {s < p.sequences ? s : -1, (t - s * tiles) * per, {s * n, n}};
    }
    unsigned before = 0;
    for (int s0 = 0; s0 < p.sequences; s0 += 64) {
        const int left = p.sequences - s0;
        const Rows r = rows_of(p, s0 + (lane < left ? lane : left - 1));
        const unsigned own = lane >= left ? 0 : r.count > per ? (r.count + per - 1) / per : 1;
        unsigned end = own;
        for (int d = 1; d < min(left, 64); d <<= 1) {
            const unsigned o = __shfl_up(end, d);
            end += lane >= d ? o : 0;
        }
        const unsigned long long hit = __ballot(lane < left && (unsigned)t < before + end);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            const unsigned nth = t - before - __builtin_amdgcn_readlane(end - own, l);
            // starts that overlap may count more tiles than 32 bits hold
            if (nth >= (unsigned)__builtin_amdgcn_readlane(own, l)) break;
            return {s0 + l, (int)nth * per,
                    {__builtin_amdgcn_readlane(r.first, l), __builtin_amdgcn_readlane(r.count, l)}};
        }
        before += __builtin_amdgcn_readlane(end, min(left, 64) - 1);
    }
    return {-1, 0, {0, 0}};
}
// at least as many tiles as there are
inline size_t tile_count(const Sequences &p, size_t per) {
    if (!p.starts) {
        const size_t n = (size_t)p.tokens / p.sequences;
        return p.sequences * (n > per ? (n + per - 1) / per : 1);
    }
    return p.tokens / per + p.sequences;
}

// Where a sequence's state comes from and goes: a slot, or none.
constexpr int kNoState = -1, kBadState = -2;
__device__ __forceinline__ int slot_in(const Sequences &p, int s) {
    const int i = p.slots_in ? p.slots_in[s] : -1;
    return i < 0 ? kNoState : i < p.slots ? i : kBadState;
}
__device__ __forceinline__ int slot_out(const Sequences &p, int s) {
    const int i = p.slots_out ? p.slots_out[s] : -1;
    return i >= 0 && i < p.slots ? i : kNoState;
}

}  // namespace exl3k

// exl3_short_conv.hip -- causal depthwise convolution of packed sequences, with their states.
//
// y_i = silu(bias + sum_j w_j x_(i - W + 1 + j)).  Bound by the rows' bytes.  A thread takes C channels of a tile of
// rows of one sequence and keeps the last W - 1 rows in registers; four rows are on their way while the four ahead of
// them are worked on.  The rows ahead of a sequence's first come from its state, and only the
// threads of its first tile read that state: they also write the one that it leaves, so a slot may be both.
// 8192 rows of 6144 fp16 channels, W = 4 with silu: 44.4 us, 4.5 TB/s (without the four rows ahead 46 us, with a
// branch for silu at each element 47 us).  A row each of eight sequences: 4.2 to 4.7 us (weights not through LDS: 4.9 us).
#include "exl3_activation.hpp"
#include "exl3_head_rows.hpp"
#include "exl3_packed_rows.hpp"

namespace exl3k {

namespace {

constexpr int kConvThreads = 256;

template <int F16, int C>
__device__ __forceinline__ void load_channels(const void *p, size_t at, float (&v)[C]) {
    if constexpr (C == 8) load_run8<F16>(p, at, 1, v);
    else v[0] = F16 ? (float)((const _Float16 *)p)[at] : ((const float *)p)[at];
}
template <int F16, int C>
__device__ __forceinline__ void store_channels(void *p, size_t at, const float (&v)[C]) {
    if constexpr (C == 8) store_run8<F16>(p, at, 1, v);
    else if constexpr (F16) ((_Float16 *)p)[at] = (_Float16)v[0];
    else ((float *)p)[at] = v[0];
}

// Where piece p is: eight lanes' reads of their piece i (p = 2 W lane + i) would meet in the same banks where 2 W is 8.
template <int W>
__device__ __forceinline__ int piece_at(int p) {
    return W == 4 ? p ^ (p >> 3 & 7) : p;
}

// A row's channels as loaded; eight of fp32 are at 16-byte places, not at the 32 of their type
template <int F16, int C>
struct Loaded {
    typedef typename std::conditional<F16, _Float16, float>::type T;
    typedef T V __attribute__((ext_vector_type(C), aligned(C == 8 ? 16 : sizeof(T))));
    V v;
    __device__ __forceinline__ void load(const void *p, size_t at) { v = *(const V *)((const T *)p + at); }
    __device__ __forceinline__ void to(float (&x)[C]) const {
#pragma unroll
        for (int e = 0; e < C; ++e) x[e] = (float)v[e];
    }
};

// blockIdx.x = tile * channel blocks + channel block; `per` rows a tile, at least W - 1
template <int W, int C, int XF16, int YF16>
__global__ __launch_bounds__(kConvThreads) void short_conv_kernel(ConvArgs a, int per, unsigned channel_blocks) {
    const unsigned tile = blockIdx.x / channel_blocks;
    const int c = (int)((blockIdx.x - tile * channel_blocks) * kConvThreads + threadIdx.x) * C;
    const Tile t = find_tile(a.s, (int)tile, per, threadIdx.x & 63);
    if (t.s < 0) return;
    float w[C][W], bias[C];
    if constexpr (C == 8) {
        // A wave's weights are one run of memory: they are loaded as such, and LDS gives each lane its 2 W pieces of 16
        // bytes (loaded by the lanes that need them, a load touches 64 lines).  Lanes behind the last channel take the last piece.
        __shared__ __attribute__((aligned(16))) f4 pieces[kConvThreads / 64][64 * 2 * W];
        const int lane = threadIdx.x & 63, most = a.channels / 4 * W - 1, first_piece = (c - 8 * lane) / 4 * W;
        f4 *const own = pieces[threadIdx.x >> 6];
        f4 x[2 * W];
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) x[i] = ((const f4 *)a.weight)[min(first_piece + 64 * i + lane, most)];
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) own[piece_at<W>(64 * i + lane)] = x[i];
        asm volatile("" ::: "memory");  // the wave's own
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) x[i] = own[piece_at<W>(2 * W * lane + i)];
        if (c >= a.channels) return;
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int j = 0; j < W; ++j) w[e][j] = x[(e * W + j) / 4][(e * W + j) % 4];
    } else {
        if (c >= a.channels) return;
#pragma unroll
        for (int j = 0; j < W; ++j) w[0][j] = a.weight[(size_t)c * W + j];
    }
#pragma unroll
    for (int e = 0; e < C; ++e) bias[e] = 0.f;
    if (a.bias) load_channels<0, C>(a.bias, c, bias);

    float last[W - 1][C];  // the rows ahead of the next one, the oldest first
    const size_t first = t.rows.first;
    if (t.row0 == 0) {
        const int in = slot_in(a.s, t.s), out = slot_out(a.s, t.s);
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
#pragma unroll
            for (int e = 0; e < C; ++e) last[j][e] = in == kBadState ? __builtin_nanf("") : 0.f;
            if (in >= 0) load_channels<XF16, C>(a.states, ((size_t)in * (W - 1) + j) * a.channels + c, last[j]);
        }
        if (out >= 0) {
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
                const int row = t.rows.count - (W - 1) + j;
                float v[C];
                if (row >= 0) {
                    load_channels<XF16, C>(a.x, (first + row) * a.x_stride + c, v);
                } else {
#pragma unroll
                    for (int e = 0; e < C; ++e) {
                        v[e] = 0.f;
#pragma unroll
                        for (int i = 0; i < W - 1; ++i) v[e] = i == W - 1 + row ? last[i][e] : v[e];
                    }
                }
                store_channels<XF16, C>(a.states, ((size_t)out * (W - 1) + j) * a.channels + c, v);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
            load_channels<XF16, C>(a.x, (first + t.row0 - (W - 1) + j) * a.x_stride + c, last[j]);
    }

    const auto step = [&](int row, const Loaded<XF16, C> &loaded) {
        float x[C];
        loaded.to(x);
        float y[C];
#pragma unroll
        for (int e = 0; e < C; ++e) {
            y[e] = bias[e];
#pragma unroll
            for (int j = 0; j < W - 1; ++j) y[e] = __builtin_fmaf(w[e][j], last[j][e], y[e]);
            y[e] = __builtin_fmaf(w[e][W - 1], x[e], y[e]);
#pragma unroll
            for (int j = 0; j + 1 < W - 1; ++j) last[j][e] = last[j + 1][e];
            last[W - 2][e] = x[e];
        }
        if (a.silu) {  // one branch a row: eight chains of instructions side by side
#pragma unroll
            for (int e = 0; e < C; ++e) y[e] = silu_f32(y[e]);
        }
        store_channels<YF16, C>(a.y, (first + row) * a.y_stride + c, y);
    };
    constexpr int U = 4;  // rows whose loads are on the way at once
    const int end = min(t.row0 + per, t.rows.count);
    int row = t.row0;
    if (row + U <= end) {
        Loaded<XF16, C> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u].load(a.x, (first + row + u) * a.x_stride + c);
        for (; row + 2 * U <= end; row += U) {
            Loaded<XF16, C> next[U];
#pragma unroll
            for (int u = 0; u < U; ++u) next[u].load(a.x, (first + row + U + u) * a.x_stride + c);
#pragma unroll
            for (int u = 0; u < U; ++u) step(row + u, x[u]);
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = next[u];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) step(row + u, x[u]);
        row += U;
    }
    if (row < end) {
        Loaded<XF16, C> x[U - 1];
#pragma unroll
        for (int u = 0; u < U - 1; ++u)
            if (row + u < end) x[u].load(a.x, (first + row + u) * a.x_stride + c);
#pragma unroll
        for (int u = 0; u < U - 1; ++u)
            if (row + u < end) step(row + u, x[u]);
    }
}

template <int W, int C, int XF16, int YF16>
hipError_t launch_tiles(const ConvArgs &a, hipStream_t stream) {
    const unsigned channel_blocks = (a.channels + kConvThreads * C - 1) / (kConvThreads * C);
    // Long tiles read their W - 1 rows ahead less often, short ones fill the card: 640 workgroups, 2.5 a CU.  fp16 in
    // tiles of 4, 8, 16, 32, the rule's first: 8192 rows of 6144 channels 36.6 us (50.8, 42.8, 39.9, 36.4), 2000 rows
    // 14.2 us (15.5, 14.0, 15.0, 15.4); of 1531 channels, one a thread, 1760 rows 5.6 us (6.6, 6.0, 5.6, 6.5), 3800
    // rows 8.5 us (11.1, 9.4, 8.3, 8.5), 8000 rows 12.5 us (19.7, 15.9, 12.9, 12.5).  fp32: 3800 rows of 1531 9.8 us
    // (11.9, 10.8, 9.9, 9.8); the rule loses most at 3800 rows of 1536, 12.5 us (12.6, 11.5, 10.8, 14.6).
    int per = 32;
    while (per > 4 && tile_count(a.s, per) * channel_blocks < 640) per /= 2;
    const size_t blocks = tile_count(a.s, per) * channel_blocks;
    short_conv_kernel<W, C, XF16, YF16><<<dim3((unsigned)blocks), dim3(kConvThreads), 0, stream>>>(a, per, channel_blocks);
    return hipGetLastError();
}
template <int W, int C>
hipError_t launch_types(const ConvArgs &a, int x_f16, int y_f16, hipStream_t stream) {
    if (x_f16) return y_f16 ? launch_tiles<W, C, 1, 1>(a, stream) : launch_tiles<W, C, 1, 0>(a, stream);
    return y_f16 ? launch_tiles<W, C, 0, 1>(a, stream) : launch_tiles<W, C, 0, 0>(a, stream);
}
template <int W>
hipError_t launch_width(const ConvArgs &a, int x_f16, int y_f16, hipStream_t stream) {
    return a.vec ? launch_types<W, 8>(a, x_f16, y_f16, stream) : launch_types<W, 1>(a, x_f16, y_f16, stream);
}

}  // namespace

hipError_t launch_short_conv(const ConvArgs &a, int x_f16, int y_f16, hipStream_t stream) {
    if (a.width == 2) return launch_width<2>(a, x_f16, y_f16, stream);
    if (a.width == 3) return launch_width<3>(a, x_f16, y_f16, stream);
    return launch_width<4>(a, x_f16, y_f16, stream);
}

}  // namespace exl3k

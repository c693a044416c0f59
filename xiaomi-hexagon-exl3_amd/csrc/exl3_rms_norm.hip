// exl3_rms_norm.hip -- root-mean-square norm of rows, with the residual's addition or a gate.
//
// y = w h / sqrt(mean(h^2) + eps) (times silu(gate)), h = x + residual.  Bound by the rows' bytes: a row is
// read once into registers, summed, and written from them.  L lanes hold a row, NV runs of eight elements each.
// 16,384 rows of 2048 with the residual's addition (403 MB): 71 us, 5.6 TB/s; 19,792 gated rows of 128: 5.2 us, of
// which a launch takes 4.
#include "exl3_activation.hpp"
#include "exl3_head_rows.hpp"
#include "exl3_linear_attention.hpp"

namespace exl3k {

namespace {

constexpr int kNormThreads = 256;

// Eight elements as loaded, one or two 16-byte words.
struct Run {
    u4 a, b;
};
__device__ __forceinline__ Run load_run(const void *p, size_t at, int f16) {
    Run r{};
    if (f16) {
        r.a = *(const u4 *)((const _Float16 *)p + at);
    } else {
        r.a = ((const u4 *)((const float *)p + at))[0];
        r.b = ((const u4 *)((const float *)p + at))[1];
    }
    return r;
}
__device__ __forceinline__ float run_element(const Run &r, int f16, int e) {
    if (f16) return (float)bitcast<h8>(r.a)[e];
    return e < 4 ? bitcast<f4>(r.a)[e] : bitcast<f4>(r.b)[e - 4];
}

__device__ __forceinline__ float load_one(const void *p, size_t at, int f16) {
    return f16 ? (float)((const _Float16 *)p)[at] : ((const float *)p)[at];
}
__device__ __forceinline__ void store_one(void *p, size_t at, int f16, float v) {
    if (f16) ((_Float16 *)p)[at] = (_Float16)v;
    else ((float *)p)[at] = v;
}

// row = token * heads + head; a 64-bit division only where the rows need one
struct Place {
    size_t token, head;
};
__device__ __forceinline__ Place place_of(size_t row, size_t rows, int heads) {
    if (heads == 1) return {row, 0};
    const size_t token = rows >> 32 ? row / heads : (uint32_t)row / (uint32_t)heads;
    return {token, row - token * heads};
}

// sum over the L lanes of a row; a row of the whole workgroup goes through LDS
template <int L>
__device__ __forceinline__ float lanes_sum(float v, float *lds) {
    v += dpp_xor<1>(v);
    v += dpp_xor<2>(v);
    v += dpp_xor<4>(v);
    if constexpr (L > 8) v += dpp_xor<8>(v);
    if constexpr (L > 16) v += __shfl_xor(v, 16);
    if constexpr (L > 32) v += __shfl_xor(v, 32);
    if constexpr (L > 64) {
        __syncthreads();  // the row before has been read
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    }
    return v;
}

template <int L, int NV>
__global__ __launch_bounds__(kNormThreads) void rms_norm_kernel(NormArgs a) {
    __shared__ float lds[4];
    const int l = threadIdx.x % L;
    const size_t rows = a.tokens * a.x.heads, per = kNormThreads / L;
    const float inv_width = 1.0f / (float)a.width;
    float w[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = 8 * (l + i * L);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[i][e] = 1.f;
        if (a.weight && at < a.width) load_run8<0>(a.weight, at, 1, w[i]);
    }
    // whole workgroups step together: every lane takes part in the sums
    for (size_t row0 = (size_t)blockIdx.x * per; row0 < rows; row0 += (size_t)gridDim.x * per) {
        const size_t row = row0 + threadIdx.x / L;
        const auto [token, head] = place_of(row, rows, a.x.heads);
        const bool in = row < rows;
        Run x[NV], r[NV], z[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = 8 * (l + i * L);
            x[i] = r[i] = z[i] = Run{};
            if (!in || at >= a.width) continue;
            x[i] = load_run(a.x.data, token * a.x.token_stride + head * a.x.head_stride + at, a.x_f16);
            if (a.res.data)
                r[i] = load_run(a.res.data, token * a.res.token_stride + head * a.res.head_stride + at, a.res_f16);
            if (a.gate.data)
                z[i] = load_run(a.gate.data, token * a.gate.token_stride + head * a.gate.head_stride + at, a.x_f16);
        }
        float h[NV][8], sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                h[i][e] = run_element(x[i], a.x_f16, e);
                if (a.res.data) h[i][e] += run_element(r[i], a.res_f16, e);
                sum = __builtin_fmaf(h[i][e], h[i][e], sum);
            }
        }
        const float s = inverse_root(__builtin_fmaf(lanes_sum<L>(sum, lds), inv_width, a.eps));
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int at = 8 * (l + i * L);
            if (!in || at >= a.width) continue;
            if (a.res_out.data) {
                const size_t to = token * a.res_out.token_stride + head * a.res_out.head_stride + at;
                if (a.res_f16) store_run8<1>(a.res_out.data, to, 1, h[i]);
                else store_run8<0>(a.res_out.data, to, 1, h[i]);
            }
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y[e] = h[i][e] * s * w[i][e];
                if (a.gate.data) y[e] *= silu_f32(run_element(z[i], a.x_f16, e));
            }
            const size_t to = token * a.out.token_stride + head * a.out.head_stride + at;
            if (a.y_f16) store_run8<1>(a.out.data, to, 1, y);
            else store_run8<0>(a.out.data, to, 1, y);
        }
    }
}

// Rows of any width and alignment, element by element: a workgroup keeps the first kHeld elements a lane in
// registers and reads those beyond twice, the second time from the caches.  Each element is read and written by
// one lane, so that a row may be normed in place.  777 rows of 1531 elements: 5.7 us (with a wait at each
// element 7.4 us, read twice 9.4 us).
constexpr int kHeld = 8;
// All loads are on their way before the first is waited for; lanes behind the row's end load its last element.
template <typename T>
__device__ __forceinline__ void load_held(const void *p, size_t at, int width, float (&v)[kHeld]) {
    T x[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) x[j] = ((const T *)p)[at + min((int)threadIdx.x + j * kNormThreads, width - 1)];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) v[j] = (float)x[j];
}
__device__ __forceinline__ void load_held(const void *p, size_t at, int f16, int width, float (&v)[kHeld]) {
    if (f16) load_held<_Float16>(p, at, width, v);
    else load_held<float>(p, at, width, v);
}
__global__ __launch_bounds__(kNormThreads) void rms_norm_any_kernel(NormArgs a) {
    __shared__ float lds[4];
    const size_t rows = a.tokens * a.x.heads;
    float w[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) w[j] = 1.f;
    if (a.weight) load_held<float>(a.weight, 0, a.width, w);
    for (size_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const auto [token, head] = place_of(row, rows, a.x.heads);
        const size_t xa = token * a.x.token_stride + head * a.x.head_stride;
        const size_t ra = token * a.res.token_stride + head * a.res.head_stride;
        const size_t za = token * a.gate.token_stride + head * a.gate.head_stride;
        const size_t qa = token * a.res_out.token_stride + head * a.res_out.head_stride;
        const size_t ya = token * a.out.token_stride + head * a.out.head_stride;
        float h[kHeld], more[kHeld] = {}, z[kHeld] = {}, sum = 0.f;
        load_held(a.x.data, xa, a.x_f16, a.width, h);
        if (a.res.data) load_held(a.res.data, ra, a.res_f16, a.width, more);
        if (a.gate.data) load_held(a.gate.data, za, a.x_f16, a.width, z);
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            if (a.res.data) h[j] += more[j];
            if ((int)threadIdx.x + j * kNormThreads < a.width) sum = __builtin_fmaf(h[j], h[j], sum);
        }
        const auto element = [&](int i) {
            float v = load_one(a.x.data, xa + i, a.x_f16);
            if (a.res.data) v += load_one(a.res.data, ra + i, a.res_f16);
            return v;
        };
        for (int i = threadIdx.x + kHeld * kNormThreads; i < a.width; i += kNormThreads) {
            const float v = element(i);
            sum = __builtin_fmaf(v, v, sum);
        }
        const float s = inverse_root(__builtin_fmaf(lanes_sum<kNormThreads>(sum, lds), 1.0f / (float)a.width, a.eps));
        const auto write = [&](int i, float v, float weight, float gate) {
            if (a.res_out.data) store_one(a.res_out.data, qa + i, a.res_f16, v);
            float y = v * s * weight;
            if (a.gate.data) y *= silu_f32(gate);
            store_one(a.out.data, ya + i, a.y_f16, y);
        };
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int i = threadIdx.x + j * kNormThreads;
            if (i < a.width) write(i, h[j], w[j], z[j]);
        }
        for (int i = threadIdx.x + kHeld * kNormThreads; i < a.width; i += kNormThreads)
            write(i, element(i), a.weight ? a.weight[i] : 1.f, a.gate.data ? load_one(a.gate.data, za + i, a.x_f16) : 0.f);
    }
}

template <int L, int NV>
hipError_t launch_rows(const NormArgs &a, hipStream_t stream) {
    const unsigned blocks = row_blocks(a.tokens * a.x.heads, kNormThreads / L);
    rms_norm_kernel<L, NV><<<dim3(blocks), dim3(kNormThreads), 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rms_norm(const NormArgs &a, hipStream_t stream) {
    const int runs = a.width / 8;
    if (!a.vec || runs > 8 * kNormThreads) {
        rms_norm_any_kernel<<<dim3(row_blocks(a.tokens * a.x.heads, 1)), dim3(kNormThreads), 0, stream>>>(a);
        return hipGetLastError();
    }
    // As few lanes as hold a row with one run each, up to a wave; beyond that a workgroup, for its shorter way from the
    // first load to the last store (4096 rows of 1024 elements: 10.0 us, a wave with two runs a lane 11.3 us; 1024
    // of 2048: 6.5 and 8.0 us; of 512, one wave 6.8, a workgroup 7.9 us; of 128, 16 lanes 5.2, 32 lanes 7.7 us).
    if (runs <= 8) return launch_rows<8, 1>(a, stream);
    if (runs <= 16) return launch_rows<16, 1>(a, stream);
    if (runs <= 32) return launch_rows<32, 1>(a, stream);
    if (runs <= 64) return launch_rows<64, 1>(a, stream);
    if (runs <= 256) return launch_rows<256, 1>(a, stream);
    if (runs <= 512) return launch_rows<256, 2>(a, stream);
    if (runs <= 1024) return launch_rows<256, 4>(a, stream);
    return launch_rows<256, 8>(a, stream);
}

}  // namespace exl3k

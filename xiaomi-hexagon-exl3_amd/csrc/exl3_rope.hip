// exl3_rope.hip -- norms and rotary positions of queries and keys in one pass.
//
// y = x / sqrt(mean(x^2) + eps) * weight, then each pair (a, b) turned by position * frequency.  Bound by
// the rows' bytes, each read and written once: D / 8 lanes hold a row, its pairs meet by lane exchange or
// within a lane, and the sines are worked out in the kernel (a table would be read as often as the rows).
// 8,192 tokens, 32 / 8 heads of 128 in fp16 (168 MB): 44 us a call over buffers in turn (3.8 TB/s), 35 us over
// the same ones, which the 256 MB cache holds (30 us in a kernel trace); one token: 3.1 us, a launch and two dependent
// round trips.
#include "exl3_head_rows.hpp"

namespace exl3k {

namespace {

constexpr int kRopeThreads = 256;

// sin and cos of position * frequency.  The frequency in turns is f * (1 / 2 pi), kept as two
// binary32 words (together 48 bits), and position * high word as its rounded product
// and the product's error (one fma), so the turn modulo 1 is good to about 2^-24 whatever the
// position: the plain binary32 product is off by 2^-24 of the whole angle, 4e-3 at
// position 65,536.  v_sin / v_cos take turns.
struct Turn {
    float hi, lo;
};
__device__ __forceinline__ Turn turn_of(float f) {
    constexpr double inv = 0.15915494309189533577;
    constexpr float inv_hi = (float)inv;
    constexpr float inv_lo = (float)(inv - (double)inv_hi);
    Turn t;
    t.hi = f * inv_hi;
    t.lo = __builtin_fmaf(f, inv_lo, __builtin_fmaf(f, inv_hi, -t.hi));
    return t;
}
__device__ __forceinline__ void sin_cos_at(Turn f, float pos, float scale, float &s, float &c) {
    const float p = pos * f.hi;
    const float err = __builtin_fmaf(pos, f.hi, -p);
    const float r = (p - __builtin_rintf(p)) + __builtin_fmaf(pos, f.lo, err);
    s = __builtin_amdgcn_sinf(r) * scale;
    c = __builtin_amdgcn_cosf(r) * scale;
}

// sum over the VL lanes of a row
template <int VL>
__device__ __forceinline__ float row_sum(float v) {
    v += dpp_xor<1>(v);
    v += dpp_xor<2>(v);
    v += dpp_xor<4>(v);
    if constexpr (VL > 8) v += dpp_xor<8>(v);
    if constexpr (VL > 16) v += __shfl_xor(v, 16);
    return v;
}

// VL lanes (head_dim / 8 rounded up to 8, 16 or 32) hold one head's row, eight elements each.
// A lane group takes one token's heads slice, slice + slices, ..: the token's sines and
// cosines are computed once for all of them.
template <int VL, int XF16, int YF16, int PAIRS>
__global__ __launch_bounds__(kRopeThreads) void qk_norm_rope_kernel(RopeArgs a, int slices) {
    const int lane = threadIdx.x & 63, l = lane & (VL - 1);
    const bool on = 8 * l < a.head_dim;  // the others only take part in the exchanges
    const int half = a.rot_dim / 2;
    const size_t units = a.tokens * slices;
    const float inv_dim = 1.0f / (float)a.head_dim;
    for (size_t unit = (size_t)blockIdx.x * (kRopeThreads / VL) + threadIdx.x / VL; unit < units;
         unit += (size_t)gridDim.x * (kRopeThreads / VL)) {  // whole lane groups
        const size_t token = unit / slices;
        const int slice = (int)(unit - token * slices);

        constexpr int NP = PAIRS ? 4 : 8;
        float sn[NP], cs[NP];
        const bool turned = on && 8 * l < a.rot_dim;
        const bool upper = !PAIRS && 8 * l >= half;
        const int partner = (lane & ~(VL - 1)) + (upper ? l - half / 8 : l + half / 8);
        if (turned) {
            const float pos = (float)a.positions[token];
            const int p0 = PAIRS ? 4 * l : (upper ? 8 * l - half : 8 * l);
    #pragma unroll
            for (int e = 0; e < NP; ++e) sin_cos_at(turn_of(a.inv_freq[p0 + e]), pos, a.rope_scale, sn[e], cs[e]);
            if (upper) {
    #pragma unroll
                for (int e = 0; e < NP; ++e) sn[e] = -sn[e];
            }
        }
        const int heads = a.q.heads + a.k.heads;
        for (int h = slice; h < heads; h += slices) {
            const bool is_q = h < a.q.heads;
            const Heads &in = is_q ? a.q : a.k;
            const Heads &out = is_q ? a.q_out : a.k_out;
            const float *w = is_q ? a.q_weight : a.k_weight;
            const int hh = is_q ? h : h - a.q.heads;
            float v[8] = {};
            if (on) load_run8<XF16>(in.data, token * in.token_stride + hh * in.head_stride + 8 * l, in.vec, v);
            if (w) {
                float sum = 0.f;
    #pragma unroll
                for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(v[e], v[e], sum);
                // v_rsq_f32 is good to 1 ulp, of normal numbers
                const float mean = __builtin_fmaf(row_sum<VL>(sum), inv_dim, a.eps);
                const bool tiny = mean < 0x1p-100f;
                const float r = __builtin_amdgcn_rsqf(tiny ? mean * 0x1p64f : mean) * (tiny ? 0x1p32f : 1.f);
                if (on) {
                    float wt[8];
                    load_run8<0>(w, 8 * l, 0, wt);
    #pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = v[e] * r * wt[e];
                }
            }
            if (a.rot_dim) {
                if constexpr (PAIRS) {
                    if (turned) {
    #pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = v[2 * e], y = v[2 * e + 1];
                            v[2 * e] = __builtin_fmaf(x, cs[e], -(y * sn[e]));
                            v[2 * e + 1] = __builtin_fmaf(y, cs[e], x * sn[e]);
                        }
                    }
                } else {
                    float o[8];
    #pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] = __shfl(v[e], partner & 63);
                    if (turned) {
    #pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(v[e], cs[e], -(o[e] * sn[e]));
                    }
                }
            }
            if (on) store_run8<YF16>(out.data, token * out.token_stride + hh * out.head_stride + 8 * l, out.vec, v);
        }
    }
}

template <int VL, int XF16, int YF16>
hipError_t launch_vl(const RopeArgs &a, hipStream_t stream) {
    // enough lane groups for every wave slot of the chip (256 CUs, 32 waves) where the heads allow it
    const size_t groups = (size_t)256 * 32 * 64 / VL;
    const int heads = a.q.heads + a.k.heads;
    size_t slices = (groups + a.tokens - 1) / a.tokens;
    slices = slices < (size_t)heads ? slices : (size_t)heads;
    const unsigned blocks = row_blocks(a.tokens * slices, kRopeThreads / VL);
    if (a.interleaved)
        qk_norm_rope_kernel<VL, XF16, YF16, 1><<<dim3(blocks), dim3(kRopeThreads), 0, stream>>>(a, (int)slices);
    else
        qk_norm_rope_kernel<VL, XF16, YF16, 0><<<dim3(blocks), dim3(kRopeThreads), 0, stream>>>(a, (int)slices);
    return hipGetLastError();
}
template <int XF16, int YF16>
hipError_t launch_types(const RopeArgs &a, hipStream_t stream) {
    if (a.head_dim <= 64) return launch_vl<8, XF16, YF16>(a, stream);
    if (a.head_dim <= 128) return launch_vl<16, XF16, YF16>(a, stream);
    return launch_vl<32, XF16, YF16>(a, stream);
}

}  // namespace

hipError_t launch_qk_norm_rope(const RopeArgs &a, int x_f16, int y_f16, hipStream_t stream) {
    if (x_f16) return y_f16 ? launch_types<1, 1>(a, stream) : launch_types<1, 0>(a, stream);
    return y_f16 ? launch_types<0, 1>(a, stream) : launch_types<0, 0>(a, stream);
}

}  // namespace exl3k

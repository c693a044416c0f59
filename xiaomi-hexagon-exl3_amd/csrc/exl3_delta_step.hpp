// exl3_delta_step.hpp -- the gated delta rule row by row: the next token(s) of many sequences.
//
//   S <- e^g S,  u = beta (v - S^T k),  S <- S + k u^T,  out = scale S^T q
//
// Bound by the states, read and written once, and with few of them by the way from row to row.
// A column of S needs nothing of the others, so a wave takes 16 columns of one head's state into
// registers, all KD rows of them: lane 4 r + c holds columns 4 c .. 4 c + 3 of the R = KD / 16 rows from r R on.
// S^T k and S^T q of the state before the row are one walk over the registers and one exchange over r, since
//   out = scale (e^g S^T q + (k . q) u).
// 16 heads of 128 x 128, one row each: 5.0 us of one sequence, of 64 sequences 25 us, 5.3 TB/s.  Waves of 32 columns
// take 7.3 and 29 us (too few on the card to hide their loads), waves of 8 columns 5.0 and 29 us (64 bytes
// of a state's row at a time).  A further row of one sequence takes 1.0 us, about 2400 cycles from k and q
// to the state; loading four rows ahead instead of one changes nothing.
#pragma once

#include "exl3_delta_gates.hpp"
#include "exl3_head_rows.hpp"

namespace exl3k {

namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));

constexpr int kStepWaves = 4;  // of a workgroup; nothing is shared

// sum over the lanes l with the same l % 4
__device__ __forceinline__ float sum_rows(float v) {
    v += dpp_xor<4>(v);
    v += dpp_xor<8>(v);
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = __int_as_float(a[0]) + __int_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return __int_as_float(b[0]) + __int_as_float(b[1]);
}

// of lane t % 64
__device__ __forceinline__ float lane_value(float v, int t) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), t & 63));
}

template <int N>
__device__ __forceinline__ void load_halves(const _Float16 *p, bool vec, _Float16 (&to)[N]) {
    typedef _Float16 hv __attribute__((ext_vector_type(N < 8 ? N : 8)));
    if (vec) {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            const hv t = *(const hv *)(p + i);
#pragma unroll
            for (int e = 0; e < (N < 8 ? N : 8); ++e) to[i + e] = t[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = p[i];
    }
}

// One row's inputs as a lane needs them: its R elements of k and q, four of v.
template <int R>
struct StepRow {
    _Float16 k[R], q[R], v[4];
};
template <int R>
__device__ __forceinline__ void load_row(const DeltaArgs &a, size_t row, int head, int kr, int col,
                                         StepRow<R> &x) {
    const int kh = head / (a.v.heads / a.k.heads);
    load_halves((const _Float16 *)a.k.data + row * a.k.token_stride + kh * a.k.head_stride + kr, a.k.vec, x.k);
    load_halves((const _Float16 *)a.q.data + row * a.q.token_stride + kh * a.q.head_stride + kr, a.q.vec, x.q);
    load_halves((const _Float16 *)a.v.data + row * a.v.token_stride + head * a.v.head_stride + col, a.v.vec, x.v);
}

// One wave's part; sequences of `limit` rows and more are left to the chunks.
template <int KD>
__device__ __forceinline__ void delta_step(const DeltaArgs &a, size_t unit, int slices, int limit) {
    constexpr int R = KD / 16;
    const int lane = threadIdx.x & 63, slice = (int)(unit % slices);
    const size_t sh = unit / slices;
    const int head = (int)(sh % a.v.heads), s = (int)(sh / a.v.heads);
    const int kr = lane / 4 * R, col = (slice * 4 + lane % 4) * 4;
    const Rows rows = rows_of(a.s, s);
    if (rows.count >= limit) return;
    const int in = slot_in(a.s, s), out = slot_out(a.s, s);
    const size_t state_size = (size_t)a.v.heads * KD * a.value_dim;
    const size_t at = ((size_t)head * KD + kr) * a.value_dim + col;

    f4 S[R];
    const float start = in == kBadState ? __builtin_nanf("") : 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        S[i] = (f4){start, start, start, start};
        if (in >= 0) S[i] = *(const f4 *)(a.states + in * state_size + at + (size_t)i * a.value_dim);
    }
    const HeadGates hg = head_gates(a, head);
    float decays = 0.f, betas = 0.f;  // of 64 rows, one a lane: far fewer instructions on the way from row to row
    StepRow<R> x, next;
    if (rows.count) load_row(a, rows.first, head, kr, col, x);
    for (int t = 0; t < rows.count; ++t) {
        const bool more = t + 1 < rows.count;
        if (more) load_row(a, (size_t)rows.first + t + 1, head, kr, col, next);
        if (t % 64 == 0) {
            const Gates gt = gates_of(a, hg, load_gates(a, (size_t)rows.first + min(t + lane, rows.count - 1), head));
            decays = decay_of(gt.g);
            betas = gt.beta;
        }
        float sk[4] = {}, sq[4] = {}, kk = 0.f, qq = 0.f, kq = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float k = (float)x.k[i], q = (float)x.q[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sk[j] = __builtin_fmaf(S[i][j], k, sk[j]);
                sq[j] = __builtin_fmaf(S[i][j], q, sq[j]);
            }
            kk = __builtin_fmaf(k, k, kk);
            qq = __builtin_fmaf(q, q, qq);
            kq = __builtin_fmaf(k, q, kq);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            sk[j] = sum_rows(sk[j]);
            sq[j] = sum_rows(sq[j]);
        }
        kq = sum_rows(kq);
        float rk = 1.f, rq = 1.f;
        if (a.eps >= 0.f) {
            rk = inverse_length(sum_rows(kk), a.eps);
            rq = inverse_length(sum_rows(qq), a.eps);
        }
        const float decay = lane_value(decays, t), beta = lane_value(betas, t);
        float u[4], o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u[j] = beta * ((float)x.v[j] - decay * rk * sk[j]);
            o[j] = a.scale * rq * (decay * sq[j] + rk * kq * u[j]);
            u[j] *= rk;
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i][j] = __builtin_fmaf((float)x.k[i], u[j], decay * S[i][j]);
        if (lane < 4) {
            _Float16 *y = (_Float16 *)a.out.data + ((size_t)rows.first + t) * a.out.token_stride +
                          head * a.out.head_stride + col;
            const h4 r = {(_Float16)o[0], (_Float16)o[1], (_Float16)o[2], (_Float16)o[3]};
            if (a.out.vec) {
                *(h4 *)y = r;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = r[j];
            }
        }
        if (more) x = next;
    }
    if (out >= 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) *(f4 *)(a.states + out * state_size + at + (size_t)i * a.value_dim) = S[i];
    }
}

}  // namespace

}  // namespace exl3k

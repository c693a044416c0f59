// exl3_delta_step.hpp -- the gated delta rule row by row: the next token(s) of many sequences.
//
//   S <- e^g S,  u = beta (v - S^T k),  S <- S + k u^T,  out = scale S^T q
//
// Bound by the states, read and written once, and with few of them by the way from row to row.
// A column of S needs nothing of the others, so a wave takes 16 columns of one head's state into
// registers, all KD rows of them: lane 4 r + c holds columns 4 c .. 4 c + 3 of the R = KD / 16 rows from r R on.
// S^T k and S^T q of the state before the row are one walk over the registers and one exchange over r, since
//   out = scale (e^g S^T q + (k . q) u).
// The sums over r of two and four numbers are exchanged together (sums_in_rows), and a row of 16 lanes works out u and out
// of one of the four columns.
// 16 heads of 128 x 128, one row each: 4.8 us of one sequence, of 64 sequences 24 us, 5.6 TB/s.  With each number
// summed by itself a further row of one sequence took 1.0 us, summed together 0.77 us, and with a row's halves kept in
// pairs, as they were loaded, 0.60 us, about 1450 cycles from k and q to the state.
// Waves of 32 columns were slower (7.3 and 29 us: too few on the card to hide their loads), waves of 8 columns
// too (5.0 and 29 us: 64 bytes of a state's row at a time); loading four rows ahead instead of one changed nothing.
#pragma once

#include "exl3_delta_gates.hpp"
#include "exl3_head_rows.hpp"

namespace exl3k {

namespace {

constexpr int kStepWaves = 4;  // of a workgroup; nothing is shared

// One of two numbers a half (32) or every second row of 16 lanes (16), summed over the pairs of halves or rows: the
// swap and the add of one sum make two.
__device__ __forceinline__ float sum_halves(float x, float y) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(y), false, false);
    return __int_as_float(a[0]) + __int_as_float(a[1]);
}
__device__ __forceinline__ float sum_row_pairs(float x, float y) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(y), false, false);
    return __int_as_float(a[0]) + __int_as_float(a[1]);
}
// Sums over the lanes l with the same l % 4: of x[0], x[2], x[1] and x[3] in rows 0, 1, 2 and 3 of 16 lanes
__device__ __forceinline__ float sums_in_rows(const float (&x)[4]) {
    float v = sum_row_pairs(sum_halves(x[0], x[1]), sum_halves(x[2], x[3]));
    v += dpp_xor<4>(v);
    return v + dpp_xor<8>(v);
}
// and back: number j of its row, for every lane
__device__ __forceinline__ void from_rows(float v, float (&x)[4]) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(a[0], a[0], false, false);
    const auto c = __builtin_amdgcn_permlane32_swap(a[1], a[1], false, false);
    x[0] = __int_as_float(b[0]);
    x[1] = __int_as_float(b[1]);
    x[2] = __int_as_float(c[0]);
    x[3] = __int_as_float(c[1]);
}

// of any lane of row r
__device__ __forceinline__ float row_value(float v, int r) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 16 * r));
}
// of lane t % 64
__device__ __forceinline__ float lane_value(float v, int t) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), t & 63));
}

// N consecutive elements, at a place of their size where `vec`
template <int N>
struct Halves {
    typedef _Float16 V __attribute__((ext_vector_type(N)));
};
template <int N>
__device__ __forceinline__ typename Halves<N>::V load_halves(const _Float16 *p, int vec) {
    typedef typename Halves<N>::V V;
    if (vec) return *(const V *)p;
    V t;
#pragma unroll
    for (int e = 0; e < N; ++e) t[e] = p[e];
    return t;
}

// One row's inputs as a lane needs them: its R elements of k and q, one of v.
template <int R>
struct StepRow {
    typename Halves<R>::V k, q;
    _Float16 v;
};
template <int R>
__device__ __forceinline__ void load_row(const DeltaArgs &a, size_t row, int head, int kr, int col,
                                         StepRow<R> &x) {
    const int kh = head / (a.v.heads / a.k.heads);
    x.k = load_halves<R>((const _Float16 *)a.k.data + row * a.k.token_stride + kh * a.k.head_stride + kr, a.k.vec);
    x.q = load_halves<R>((const _Float16 *)a.q.data + row * a.q.token_stride + kh * a.q.head_stride + kr, a.q.vec);
    x.v = ((const _Float16 *)a.v.data)[row * a.v.token_stride + head * a.v.head_stride + col];
}

// One wave's part; sequences of `limit` rows and more are left to the chunks.
template <int KD>
__device__ __forceinline__ void delta_step(const DeltaArgs &a, size_t unit, int slices, int limit) {
    constexpr int R = KD / 16;
    const int lane = threadIdx.x & 63, slice = (int)(unit % slices);
    const size_t sh = unit / slices;
    const int head = (int)(sh % a.v.heads), s = (int)(sh / a.v.heads);
    const int kr = lane / 4 * R, col = (slice * 4 + lane % 4) * 4;
    const int own = col + ((lane >> 5 & 1) | (lane >> 3 & 2));  // the column whose u and out the lane's row works out
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
    if (rows.count) load_row(a, rows.first, head, kr, own, x);
    for (int t = 0; t < rows.count; ++t) {
        const bool more = t + 1 < rows.count;
        if (more) load_row(a, (size_t)rows.first + t + 1, head, kr, own, next);
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
        const float sk_own = sums_in_rows(sk), sq_own = sums_in_rows(sq);
        const float of_row[4] = {kk, qq, kq, kq};
        const float sums = sums_in_rows(of_row);
        kq = row_value(sums, 1);
        float rk = 1.f, rq = 1.f;
        if (a.eps >= 0.f) {
            const float inverse = inverse_root(sums + a.eps);
            rk = row_value(inverse, 0);
            rq = row_value(inverse, 2);
        }
        const float decay = lane_value(decays, t), beta = lane_value(betas, t);
        const float u_own = beta * ((float)x.v - decay * rk * sk_own);
        float u[4];
        from_rows(u_own * rk, u);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i][j] = __builtin_fmaf((float)x.k[i], u[j], decay * S[i][j]);
        if ((lane & 12) == 0)
            ((_Float16 *)a.out.data)[((size_t)rows.first + t) * a.out.token_stride + head * a.out.head_stride + own] =
                (_Float16)(a.scale * rq * (decay * sq_own + rk * kq * u_own));
        if (more) x = next;
    }
    if (out >= 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) *(f4 *)(a.states + out * state_size + at + (size_t)i * a.value_dim) = S[i];
    }
}

}  // namespace

}  // namespace exl3k

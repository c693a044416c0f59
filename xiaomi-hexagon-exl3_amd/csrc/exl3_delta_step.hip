// exl3_delta_step.hip -- the gated delta rule row by row: the next token(s) of many sequences.
//
//   S <- e^g S,  u = beta (v - S^T k),  S <- S + k u^T,  out = scale S^T q
//
// Bound by the states, read and written once.  A column of S needs nothing of the others, so a wave takes
// 32 columns of one head's state into registers, all KD rows of them: lane 8 r + c holds columns 4 c .. 4 c + 3
// of rows r KD / 8 .. (r + 1) KD / 8 - 1, 128 bytes of a row a lane group.  S^T k and S^T q of the state
// before the row are one walk over the registers and one exchange over r, since
//   out = scale (e^g S^T q + (k . q) u).
#include "exl3_delta_gates.hpp"
#include "exl3_head_rows.hpp"

namespace exl3k {

namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));

// sum over lanes l, l ^ 8, l ^ 16, .. ^ 56
__device__ __forceinline__ float sum_rows(float v) {
    v += dpp_xor<8>(v);
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = __int_as_float(a[0]) + __int_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return __int_as_float(b[0]) + __int_as_float(b[1]);
}

// One row's inputs as a lane needs them: its KD / 8 elements of k and q, four of v.
template <int KD>
struct StepRow {
    float k[KD / 8], q[KD / 8], v[4], g, beta;
};
template <int KD>
__device__ __forceinline__ void load_row(const DeltaArgs &a, size_t row, int head, int kr, int col, bool on,
                                         StepRow<KD> &x) {
    const int kh = head / (a.v.heads / a.k.heads);
#pragma unroll
    for (int i = 0; i < KD / 8; i += 8) {
        load_run8<1>(a.k.data, row * a.k.token_stride + kh * a.k.head_stride + kr + i, a.k.vec,
                     *(float(*)[8]) & x.k[i]);
        load_run8<1>(a.q.data, row * a.q.token_stride + kh * a.q.head_stride + kr + i, a.q.vec,
                     *(float(*)[8]) & x.q[i]);
    }
    const _Float16 *v = (const _Float16 *)a.v.data + row * a.v.token_stride + head * a.v.head_stride + col;
    h4 t = {};
    if (on) {
        if (a.v.vec) t = *(const h4 *)v;
        else t = (h4){v[0], v[1], v[2], v[3]};
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[j] = (float)t[j];
    const Gates gt = gates_of(a, row, head);
    x.g = gt.g;
    x.beta = gt.beta;
}

template <int KD>
__global__ __launch_bounds__(256) void delta_step_kernel(DeltaArgs a, size_t units, int slices) {
    const size_t unit = (size_t)blockIdx.x * (blockDim.x / 64) + (threadIdx.x >> 6);
    if (unit >= units) return;  // a whole wave
    constexpr int R = KD / 8;
    const int lane = threadIdx.x & 63, slice = (int)(unit % slices);
    const size_t sh = unit / slices;
    const int head = (int)(sh % a.v.heads), s = (int)(sh / a.v.heads);
    const int kr = (lane >> 3) * R, col = slice * 32 + (lane & 7) * 4;
    const bool on = col < a.value_dim;
    const Rows rows = rows_of(a.s, s);
    const int in = slot_in(a.s, s), out = slot_out(a.s, s);
    const size_t state_size = (size_t)a.v.heads * KD * a.value_dim;
    const size_t at = ((size_t)head * KD + kr) * a.value_dim + col;

    f4 S[R];
    const float start = in == kBadState ? __builtin_nanf("") : 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        S[i] = (f4){start, start, start, start};
        if (in >= 0 && on) S[i] = *(const f4 *)(a.states + in * state_size + at + (size_t)i * a.value_dim);
    }
    StepRow<KD> x;
    if (rows.count) load_row<KD>(a, rows.first, head, kr, col, on, x);
    for (int t = 0; t < rows.count; ++t) {
        StepRow<KD> next;
        load_row<KD>(a, (size_t)rows.first + min(t + 1, rows.count - 1), head, kr, col, on, next);
        float sk[4] = {}, sq[4] = {}, kk = 0.f, qq = 0.f, kq = 0.f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sk[j] = __builtin_fmaf(S[i][j], x.k[i], sk[j]);
                sq[j] = __builtin_fmaf(S[i][j], x.q[i], sq[j]);
            }
            kk = __builtin_fmaf(x.k[i], x.k[i], kk);
            qq = __builtin_fmaf(x.q[i], x.q[i], qq);
            kq = __builtin_fmaf(x.k[i], x.q[i], kq);
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
        const float decay = decay_of(x.g);
        float u[4], o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u[j] = x.beta * (x.v[j] - decay * rk * sk[j]);
            o[j] = a.scale * rq * (decay * sq[j] + rk * kq * u[j]);
            u[j] *= rk;
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i][j] = __builtin_fmaf(x.k[i], u[j], decay * S[i][j]);
        if (lane < 8 && on) {
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
        x = next;
    }
    if (out >= 0 && on) {
#pragma unroll
        for (int i = 0; i < R; ++i) *(f4 *)(a.states + out * state_size + at + (size_t)i * a.value_dim) = S[i];
    }
}

}  // namespace

hipError_t launch_delta_step(const DeltaArgs &a, hipStream_t stream) {
    const int slices = (a.value_dim + 31) / 32;
    const size_t units = (size_t)a.s.sequences * a.v.heads * slices;
    const int waves = units < 2048 ? 1 : 4;
    const unsigned blocks = (unsigned)((units + waves - 1) / waves);
    if (a.key_dim == 64)
        delta_step_kernel<64><<<dim3(blocks), dim3(64 * waves), 0, stream>>>(a, units, slices);
    else
        delta_step_kernel<128><<<dim3(blocks), dim3(64 * waves), 0, stream>>>(a, units, slices);
    return hipGetLastError();
}

}  // namespace exl3k

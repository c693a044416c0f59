// exl3_linear_attention_api.cpp -- the C-ABI of the linear-attention block (include/exl3_hip.h):
// argument checks and dispatch to its gfx950 kernels.
#include "exl3_linear_attention.hpp"

#include <hip/hip_runtime.h>

#include <cmath>

#include "exl3_hip.h"
#include "exl3_views.hpp"

using namespace exl3k;

namespace {

constexpr size_t kMaxSlots = (size_t)1 << 30;

// Sequences over `tokens` rows with states of `state_bytes` bytes in a pool.
bool packed(const int32_t *starts, size_t sequences, size_t tokens, const void *states, size_t slots,
            const int32_t *slots_in, const int32_t *slots_out, size_t state_bytes, Sequences *s) {
    if (sequences > kMaxSequences || tokens > kMaxTokens || slots > kMaxSlots) return false;
    if (!starts && sequences && tokens % sequences) return false;
    if (!aligned(starts, 4) || !aligned(slots_in, 4) || !aligned(slots_out, 4) || !aligned(states, 16)) return false;
    if ((slots_in || slots_out) && (!states || !slots)) return false;
    if (slots && slots > ((size_t)1 << 50) / state_bytes) return false;  // byte offsets far below 2^64
    s->starts = starts;
    s->slots_in = slots_in;
    s->slots_out = slots_out;
    s->sequences = (int)sequences;
    s->tokens = (int)tokens;
    s->slots = (int)slots;
    return true;
}

bool delta_dims(size_t v_heads, size_t key_dim, size_t value_dim) {
    return v_heads >= 1 && v_heads <= kMaxHeads && (key_dim == 64 || key_dim == 128) && value_dim >= 16 &&
           value_dim <= 256 && value_dim % 16 == 0;
}

}  // namespace

extern "C" {

exl3_status exl3_hip_rms_norm(const exl3_head_view *x, const exl3_head_view *gate, exl3_dtype xt,
                              const exl3_head_view *residual, const exl3_head_view *residual_out, exl3_dtype rt,
                              size_t tokens, size_t width, const float *weight, float eps, const exl3_head_view *out,
                              exl3_dtype yt, hipStream_t stream) {
    if (!valid_dtype(xt) || !valid_dtype(yt) || !valid_dtype(rt) || tokens > kMaxTokens) return EXL3_INVAL_PARAMS;
    if (width < 1 || width > 65536 || !aligned(weight, 4) || !(eps >= 0.f) || !std::isfinite(eps))
        return EXL3_INVAL_PARAMS;
    if (residual_out && !residual) return EXL3_INVAL_PARAMS;
    if (!tokens) return EXL3_OK;
    NormArgs a{};
    if (!head_view(x, tokens, width, xt, false, &a.x) || !head_view(out, tokens, width, yt, true, &a.out) ||
        (gate && !head_view(gate, tokens, width, xt, false, &a.gate)) ||
        (residual && !head_view(residual, tokens, width, rt, false, &a.res)) ||
        (residual_out && !head_view(residual_out, tokens, width, rt, true, &a.res_out)))
        return EXL3_INVAL_PARAMS;
    if (a.out.heads != a.x.heads || (gate && a.gate.heads != a.x.heads) || (residual && a.res.heads != a.x.heads) ||
        (residual_out && a.res_out.heads != a.x.heads))
        return EXL3_INVAL_PARAMS;
    // in place only where the lane that reads an element writes it
    if (a.out.data == a.x.data && !(xt == yt && same_view(a.out, a.x))) return EXL3_INVAL_PARAMS;
    if ((gate && a.out.data == a.gate.data) || (residual && a.out.data == a.res.data)) return EXL3_INVAL_PARAMS;
    if (residual_out && ((a.res_out.data == a.res.data && !same_view(a.res_out, a.res)) ||
                         a.res_out.data == a.x.data || a.res_out.data == a.out.data ||
                         (gate && a.res_out.data == a.gate.data)))
        return EXL3_INVAL_PARAMS;
    a.weight = weight;
    a.tokens = tokens;
    a.width = (int)width;
    a.x_f16 = xt == EXL3_F16;
    a.res_f16 = rt == EXL3_F16;
    a.y_f16 = yt == EXL3_F16;
    a.vec = width % 8 == 0 && a.x.vec && a.out.vec && (!gate || a.gate.vec) && (!residual || a.res.vec) &&
            (!residual_out || a.res_out.vec) && aligned(weight, 16);
    a.eps = eps;
    return from_hip(launch_rms_norm(a, stream));
}

exl3_status exl3_hip_short_conv(const void *x, exl3_dtype xt, size_t x_row_stride, size_t tokens, size_t channels,
                                const float *weight, size_t width, const float *bias, int silu, const int32_t *starts,
                                size_t sequences, void *states, size_t slots, const int32_t *slots_in,
                                const int32_t *slots_out, void *y, exl3_dtype yt, size_t y_row_stride,
                                hipStream_t stream) {
    if (!valid_dtype(xt) || !valid_dtype(yt) || channels < 1 || channels > ((size_t)1 << 20) || width < 2 || width > 4)
        return EXL3_INVAL_PARAMS;
    ConvArgs a{};
    if (!packed(starts, sequences, tokens, states, slots, slots_in, slots_out, (width - 1) * channels * dtype_size(xt),
                &a.s))
        return EXL3_INVAL_PARAMS;
    if (x_row_stride < channels || y_row_stride < channels || x_row_stride > kMaxStride || y_row_stride > kMaxStride ||
        (tokens > 1 && (x_row_stride > kMaxSpan / (tokens - 1) || y_row_stride > kMaxSpan / (tokens - 1))))
        return EXL3_INVAL_PARAMS;
    if (!weight || !aligned(weight, 4) || !aligned(bias, 4) || !aligned(x, dtype_size(xt)) ||
        !aligned(y, dtype_size(yt)) || (tokens && (!x || !y || x == y)))
        return EXL3_INVAL_PARAMS;
    if (!sequences) return EXL3_OK;
    if ((tokens / 32 + sequences) * ((channels + 255) / 256) >= ((size_t)1 << 23)) return EXL3_NO_SUPPORT;
    a.x = x;
    a.y = y;
    a.states = states;
    a.weight = weight;
    a.bias = bias;
    a.x_stride = x_row_stride;
    a.y_stride = y_row_stride;
    a.channels = (int)channels;
    a.width = (int)width;
    a.silu = silu != 0;
    a.vec = channels % 8 == 0 && aligned(x, 16) && aligned(y, 16) && x_row_stride % 8 == 0 && y_row_stride % 8 == 0 &&
            aligned(weight, 16) && aligned(bias, 16);
    return from_hip(launch_short_conv(a, xt == EXL3_F16, yt == EXL3_F16, stream));
}

size_t exl3_hip_delta_rule_workspace_bytes(size_t v_heads, size_t key_dim, size_t value_dim, size_t sequences,
                                           size_t tokens) {
    if (!delta_dims(v_heads, key_dim, value_dim) || sequences > kMaxSequences || tokens > kMaxTokens || !sequences)
        return 0;
    return delta_prompt_bytes(v_heads, (int)key_dim, sequences, tokens);
}

exl3_status exl3_hip_delta_rule(const exl3_head_view *q, const exl3_head_view *k, const exl3_head_view *v,
                                const float *g, const float *beta, size_t gate_stride, const float *a_log,
                                const float *dt_bias, const exl3_head_view *out, size_t key_dim, size_t value_dim,
                                const int32_t *starts, size_t sequences, size_t tokens, float *states, size_t slots,
                                const int32_t *slots_in, const int32_t *slots_out, float scale, float qk_eps,
                                void *workspace, size_t workspace_bytes, hipStream_t stream) {
    if (!v || !delta_dims(v->heads, key_dim, value_dim)) return EXL3_INVAL_PARAMS;
    DeltaArgs a{};
    if (!packed(starts, sequences, tokens, states, slots, slots_in, slots_out, v->heads * key_dim * value_dim * 4,
                &a.s))
        return EXL3_INVAL_PARAMS;
    if (!head_view(q, tokens, key_dim, EXL3_F16, false, &a.q) || !head_view(k, tokens, key_dim, EXL3_F16, false, &a.k) ||
        !head_view(v, tokens, value_dim, EXL3_F16, false, &a.v) ||
        !head_view(out, tokens, value_dim, EXL3_F16, true, &a.out))
        return EXL3_INVAL_PARAMS;
    if (a.q.heads != a.k.heads || a.v.heads != a.out.heads || a.v.heads % a.k.heads) return EXL3_INVAL_PARAMS;
    if (tokens && (a.out.data == a.q.data || a.out.data == a.k.data || a.out.data == a.v.data)) return EXL3_INVAL_PARAMS;
    if ((tokens && (!g || !beta)) || !aligned(g, 4) || !aligned(beta, 4) || gate_stride < v->heads ||
        gate_stride > kMaxStride || (tokens > 1 && gate_stride > kMaxSpan / (tokens - 1)))
        return EXL3_INVAL_PARAMS;
    if (!a_log != !dt_bias || !aligned(a_log, 4) || !aligned(dt_bias, 4)) return EXL3_INVAL_PARAMS;
    if (!std::isfinite(scale) || !std::isfinite(qk_eps)) return EXL3_INVAL_PARAMS;
    if (!sequences) return EXL3_OK;
    if ((tokens / 64 + sequences) * v->heads * (value_dim / 16) >= ((size_t)1 << 22)) return EXL3_NO_SUPPORT;
    a.g = g;
    a.beta = beta;
    a.a_log = a_log;
    a.dt_bias = dt_bias;
    a.gate_stride = gate_stride;
    a.states = states;
    a.key_dim = (int)key_dim;
    a.value_dim = (int)value_dim;
    a.scale = scale;
    a.eps = qk_eps;
    const size_t need = delta_prompt_bytes(v->heads, a.key_dim, sequences, tokens);
    if (!need || !delta_prompt_serves(a)) return from_hip(launch_delta_step(a, stream));
    WorkspaceLease lease;
    const exl3_status st = take_workspace(need, stream, &lease, &workspace, &workspace_bytes);
    if (st != EXL3_OK) return st;
    return from_hip(launch_delta_prompt(a, workspace, stream));
}

}  // extern "C"

// exl3_attention_prompt.hip -- attention of packed sequences over their own keys and values.
#include "exl3_attention_rows.hpp"

namespace exl3k {

namespace {

struct PromptRows {
    const _Float16 *k, *v;
    size_t k_stride, v_stride;
    __device__ float key(int n, int i) const { return (float)k[n * k_stride + i]; }
    __device__ float value(int n, int i) const { return (float)v[n * v_stride + i]; }
};

// One wave per query row and head.
template <int D>
__global__ __launch_bounds__(64) void attention_prompt_kernel(PromptArgs a) {
    const int row = blockIdx.x, head = blockIdx.y;
    int s = 0;
    while (s < a.sequences && !(row >= a.q_starts[s] && row < a.q_starts[s + 1])) ++s;
    if (s == a.sequences) return;
    const int q0 = a.q_starts[s], q1 = a.q_starts[s + 1];
    int k0 = a.kv_starts[s], k1 = a.kv_starts[s + 1];
    k0 = k0 < 0 ? 0 : k0;
    k1 = k1 > a.kv_tokens ? a.kv_tokens : k1;
    const int nk = k1 > k0 ? k1 - k0 : 0;
    const int seen = a.causal ? nk - (q1 - 1 - row) : nk;
    const int kvh = head / (a.q.heads / a.k.heads);
    PromptRows r;
    r.k_stride = a.k.token_stride;
    r.v_stride = a.v.token_stride;
    r.k = (const _Float16 *)a.k.data + (size_t)k0 * r.k_stride + kvh * a.k.head_stride;
    r.v = (const _Float16 *)a.v.data + (size_t)k0 * r.v_stride + kvh * a.v.head_stride;
    float o[D / 64];
    const float inv = attend_row<D>((const _Float16 *)a.q.data + (size_t)row * a.q.token_stride + head * a.q.head_stride,
                                    0, r, seen, a.scale, o);
    (void)q0;
    _Float16 *out = (_Float16 *)a.out.data + (size_t)row * a.out.token_stride + head * a.out.head_stride;
    for (int i = 0; i < D / 64; ++i) out[i * 64 + threadIdx.x] = (_Float16)(o[i] * inv);
}

}  // namespace

hipError_t launch_attention_prompt(const PromptArgs &a, hipStream_t stream) {
    const dim3 grid(a.q_tokens, a.q.heads);
    if (a.head_dim == 64) attention_prompt_kernel<64><<<grid, 64, 0, stream>>>(a);
    else if (a.head_dim == 128) attention_prompt_kernel<128><<<grid, 64, 0, stream>>>(a);
    else attention_prompt_kernel<256><<<grid, 64, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace exl3k

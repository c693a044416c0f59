// exl3_attention_api.cpp -- the C-ABI of the attention block (include/exl3_hip.h):
// argument checks, views and dispatch to its gfx950 kernels.
#include <hip/hip_runtime.h>

#include <cmath>

#include "exl3_attention.hpp"
#include "exl3_hip.h"
#include "exl3_launch.hpp"
#include "exl3_views.hpp"

using namespace exl3k;

namespace {

constexpr size_t kMaxGroup = 64;                 // q heads per kv head
constexpr size_t kMaxGridX = ((size_t)1 << 23) - 1;  // workgroups of 512: fewer than 2^32 work-items

bool attention_dim(size_t d) { return d == 64 || d == 128 || d == 256; }

}  // namespace

extern "C" {

exl3_status exl3_hip_qk_norm_rope(const exl3_head_view *q, const exl3_head_view *k, exl3_dtype xt, size_t tokens,
                                  size_t head_dim, const float *q_weight, const float *k_weight, float eps,
                                  const int32_t *positions, const float *inv_freq, size_t rot_dim, int interleaved,
                                  float rope_scale, const exl3_head_view *q_out, const exl3_head_view *k_out,
                                  exl3_dtype yt, hipStream_t stream) {
    if (!valid_dtype(xt) || !valid_dtype(yt) || tokens > kMaxTokens) return EXL3_INVAL_PARAMS;
    if (head_dim < 8 || head_dim > 256 || head_dim % 8 || rot_dim % 16 || rot_dim > head_dim) return EXL3_INVAL_PARAMS;
    if (!tokens) return EXL3_OK;
    exl3k::RopeArgs a{};
    if (!head_view(q, tokens, head_dim, xt, false, &a.q) || !head_view(q_out, tokens, head_dim, yt, true, &a.q_out) ||
        a.q.heads != a.q_out.heads)
        return EXL3_INVAL_PARAMS;
    if (k || k_out) {
        if (!head_view(k, tokens, head_dim, xt, false, &a.k) ||
            !head_view(k_out, tokens, head_dim, yt, true, &a.k_out) || a.k.heads != a.k_out.heads)
            return EXL3_INVAL_PARAMS;
    }
    // in place only where each element is read and written by the same lane
    if ((a.q.data == a.q_out.data && !(xt == yt && same_view(a.q, a.q_out))) ||
        (a.k.data && a.k.data == a.k_out.data && !(xt == yt && same_view(a.k, a.k_out))))
        return EXL3_INVAL_PARAMS;
    if (rot_dim && (!positions || !inv_freq || !aligned(positions, 4) || !aligned(inv_freq, 4)))
        return EXL3_INVAL_PARAMS;
    if (!aligned(q_weight, 4) || !aligned(k_weight, 4) || !(eps >= 0.f)) return EXL3_INVAL_PARAMS;
    a.q_weight = q_weight;
    a.k_weight = k_weight;
    a.inv_freq = inv_freq;
    a.positions = positions;
    a.tokens = tokens;
    a.head_dim = (int)head_dim;
    a.rot_dim = (int)rot_dim;
    a.interleaved = interleaved != 0;
    a.eps = eps;
    a.rope_scale = rope_scale;
    return from_hip(exl3k::launch_qk_norm_rope(a, xt == EXL3_F16, yt == EXL3_F16, stream));
}

size_t exl3_hip_kv_page_bytes(unsigned bits, size_t kv_heads, size_t head_dim, size_t page_tokens) {
    if ((bits != 4 && bits != 8) || !attention_dim(head_dim) || kv_heads < 1 || kv_heads > kMaxHeads) return 0;
    if (page_tokens < 16 || page_tokens % 16 || page_tokens > 65536) return 0;
    return exl3k::kv_layout(bits, kv_heads, head_dim, page_tokens).page_bytes;
}

exl3_status exl3_hip_kv_cache_write(void *pages, size_t page_count, unsigned bits, size_t page_tokens, size_t head_dim,
                                    const exl3_head_view *k, const exl3_head_view *v, exl3_dtype xt, size_t tokens,
                                    const int64_t *slots, int *bad_slots, hipStream_t stream) {
    if (!valid_dtype(xt) || tokens > kMaxTokens || page_count > kMaxTokens) return EXL3_INVAL_PARAMS;
    if (!k || !exl3_hip_kv_page_bytes(bits, k->heads, head_dim, page_tokens)) return EXL3_INVAL_PARAMS;
    if (!tokens) return EXL3_OK;
    exl3k::Heads kh{}, vh{};
    if (!head_view(k, tokens, head_dim, xt, false, &kh) || !head_view(v, tokens, head_dim, xt, false, &vh) ||
        kh.heads != vh.heads)
        return EXL3_INVAL_PARAMS;
    if (!pages || !aligned(pages, 16) || !slots || !aligned(slots, 8) || !aligned(bad_slots, 4))
        return EXL3_INVAL_PARAMS;
    return from_hip(exl3k::launch_kv_write((uint8_t *)pages, page_count,
                                           exl3k::kv_layout(bits, k->heads, head_dim, page_tokens), kh, vh,
                                           xt == EXL3_F16, tokens, slots, bad_slots, stream));
}

exl3_status exl3_hip_kv_cache_read(const void *pages, size_t page_count, unsigned bits, size_t page_tokens,
                                   size_t head_dim, const int64_t *slots, size_t tokens, const exl3_head_view *k_out,
                                   const exl3_head_view *v_out, exl3_dtype yt, int *bad_slots, hipStream_t stream) {
    if (!valid_dtype(yt) || tokens > kMaxTokens || page_count > kMaxTokens) return EXL3_INVAL_PARAMS;
    if (!k_out || !exl3_hip_kv_page_bytes(bits, k_out->heads, head_dim, page_tokens)) return EXL3_INVAL_PARAMS;
    if (!tokens) return EXL3_OK;
    exl3k::Heads kh{}, vh{};
    if (!head_view(k_out, tokens, head_dim, yt, true, &kh) || !head_view(v_out, tokens, head_dim, yt, true, &vh) ||
        kh.heads != vh.heads)
        return EXL3_INVAL_PARAMS;
    if (!pages || !aligned(pages, 16) || !slots || !aligned(slots, 8) || !aligned(bad_slots, 4))
        return EXL3_INVAL_PARAMS;
    return from_hip(exl3k::launch_kv_read((const uint8_t *)pages, page_count,
                                          exl3k::kv_layout(bits, k_out->heads, head_dim, page_tokens), slots, tokens,
                                          kh, vh, yt == EXL3_F16, bad_slots, stream));
}

size_t exl3_hip_attention_cached_workspace_bytes(size_t q_heads, size_t kv_heads, size_t head_dim, size_t sequences,
                                                 size_t q_len) {
    if (!attention_dim(head_dim) || kv_heads < 1 || kv_heads > kMaxHeads || q_heads < kv_heads ||
        q_heads > kMaxHeads || q_heads % kv_heads || q_heads / kv_heads > kMaxGroup || sequences > kMaxSequences ||
        q_len < 1 || q_len > 65536 || sequences * q_len > kMaxTokens)
        return 0;
    return exl3k::attention_cached_bytes(q_heads, kv_heads, head_dim, sequences, q_len);
}

exl3_status exl3_hip_attention_cached(const exl3_head_view *q, const exl3_head_view *out, size_t head_dim,
                                      const void *pages, size_t page_count, unsigned bits, size_t page_tokens,
                                      size_t kv_heads, const int32_t *page_table, size_t table_stride,
                                      const int32_t *kv_lens, size_t sequences, size_t q_len, float scale,
                                      void *workspace, size_t workspace_bytes, hipStream_t stream) {
    if (!q || !exl3_hip_kv_page_bytes(bits, kv_heads, head_dim, page_tokens)) return EXL3_INVAL_PARAMS;
    const size_t need =
        exl3_hip_attention_cached_workspace_bytes(q->heads, kv_heads, head_dim, sequences, q_len);
    if (!need || page_count < 1 || page_count > kMaxTokens || table_stride < 1 ||
        table_stride > kMaxTokens / page_tokens)
        return EXL3_INVAL_PARAMS;
    if (!sequences) return EXL3_OK;
    exl3k::CachedArgs a{};
    const size_t rows = sequences * q_len;
    if (!head_view(q, rows, head_dim, EXL3_F16, false, &a.q) ||
        !head_view(out, rows, head_dim, EXL3_F16, true, &a.out) || a.q.heads != a.out.heads ||
        a.q.data == a.out.data)
        return EXL3_INVAL_PARAMS;
    if (!pages || !aligned(pages, 16) || !page_table || !aligned(page_table, 4) || !kv_lens || !aligned(kv_lens, 4))
        return EXL3_INVAL_PARAMS;
    if (!std::isfinite(scale)) return EXL3_INVAL_PARAMS;  // the kernels bound it from below, which a NaN would pass
    if (!exl3k::attention_cached_fits(q->heads, kv_heads, sequences, q_len)) return EXL3_NO_SUPPORT;
    exl3k::WorkspaceLease lease;
    const exl3_status st = exl3k::take_workspace(need, stream, &lease, &workspace, &workspace_bytes);
    if (st != EXL3_OK) return st;
    a.pages = (const uint8_t *)pages;
    a.page_count = page_count;
    a.table_stride = table_stride;
    a.l = exl3k::kv_layout(bits, kv_heads, head_dim, page_tokens);
    a.page_table = page_table;
    a.kv_lens = kv_lens;
    a.sequences = (int)sequences;
    a.q_len = (int)q_len;
    a.scale = scale;
    return from_hip(exl3k::launch_attention_cached(a, workspace, stream));
}

size_t exl3_hip_attention_prompt_workspace_bytes(size_t q_heads, size_t head_dim, size_t sequences, size_t q_tokens,
                                                 size_t kv_tokens) {
    if (!attention_dim(head_dim) || q_heads < 1 || q_heads > kMaxHeads || sequences > kMaxSequences ||
        q_tokens > kMaxTokens || kv_tokens > kMaxTokens || !sequences || !q_tokens)
        return 0;
    return exl3k::attention_prompt_bytes(q_heads, (int)head_dim, (int)sequences, (int)q_tokens, (int)kv_tokens);
}

exl3_status exl3_hip_attention_prompt(const exl3_head_view *q, const exl3_head_view *k, const exl3_head_view *v,
                                      const exl3_head_view *out, size_t head_dim, const int32_t *q_starts,
                                      const int32_t *kv_starts, size_t sequences, size_t q_tokens, size_t kv_tokens,
                                      float scale, int causal, void *workspace, size_t workspace_bytes,
                                      hipStream_t stream) {
    if (!attention_dim(head_dim) || sequences > kMaxSequences || q_tokens > kMaxTokens || kv_tokens > kMaxTokens)
        return EXL3_INVAL_PARAMS;
    if (!sequences || !q_tokens) return EXL3_OK;
    exl3k::PromptArgs a{};
    if (!head_view(q, q_tokens, head_dim, EXL3_F16, false, &a.q) ||
        !head_view(k, kv_tokens, head_dim, EXL3_F16, false, &a.k) ||
        !head_view(v, kv_tokens, head_dim, EXL3_F16, false, &a.v) ||
        !head_view(out, q_tokens, head_dim, EXL3_F16, true, &a.out))
        return EXL3_INVAL_PARAMS;
    if (a.q.heads != a.out.heads || a.k.heads != a.v.heads || a.q.heads % a.k.heads || a.out.data == a.q.data ||
        a.out.data == a.k.data || a.out.data == a.v.data)
        return EXL3_INVAL_PARAMS;
    if (!q_starts || !kv_starts || !aligned(q_starts, 4) || !aligned(kv_starts, 4)) return EXL3_INVAL_PARAMS;
    if (!std::isfinite(scale)) return EXL3_INVAL_PARAMS;
    if ((q_tokens / 128 + sequences) * q->heads > kMaxGridX) return EXL3_NO_SUPPORT;
    a.q_starts = q_starts;
    a.kv_starts = kv_starts;
    a.head_dim = (int)head_dim;
    a.sequences = (int)sequences;
    a.q_tokens = (int)q_tokens;
    a.kv_tokens = (int)kv_tokens;
    a.causal = causal != 0;
    a.scale = scale;
    const size_t need = exl3k::attention_prompt_bytes(q->heads, a.head_dim, a.sequences, a.q_tokens, a.kv_tokens);
    exl3k::WorkspaceLease lease;
    if (need) {
        const exl3_status st = exl3k::take_workspace(need, stream, &lease, &workspace, &workspace_bytes);
        if (st != EXL3_OK) return st;
    }
    return from_hip(exl3k::launch_attention_prompt(a, need ? workspace : nullptr, stream));
}

}  // extern "C"

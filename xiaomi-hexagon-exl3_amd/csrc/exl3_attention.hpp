// exl3_attention.hpp -- internal interface between the attention block's C-ABI
// (exl3_attention_api.cpp) and its gfx950 kernels (exl3_rope.hip, exl3_kv_cache.hip,
// exl3_attention_{cached,prompt}.hip).  Launchers assume validated arguments; they only
// enqueue work and return hipGetLastError().
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "exl3_hip.h"
#include "exl3_workspace.hpp"

namespace exl3k {

// The caller's workspace checked, or the internal one of this device and stream
// (exl3_api.cpp), which the lease holds until the call's launches are enqueued.
exl3_status take_workspace(size_t need, hipStream_t stream, WorkspaceLease *lease, void **workspace, size_t *bytes);

// A view of heads inside a kernel (exl3_head_view).
struct Heads {
    void *data;
    size_t token_stride, head_stride;
    int heads;
    int vec;  // every 8-element run of a head is 16-byte aligned
};

constexpr int kKvGroup = 32;  // elements that share a scale

// Where a page's parts are (include/exl3_hip.h): for each head, from its region's start.
struct KvLayout {
    size_t page_bytes, region;  // region: one head's bytes of a page
    size_t v_off, ks_off, vs_off;
    int page_tokens, kv_heads, head_dim, bits;
};
inline KvLayout kv_layout(unsigned bits, size_t kv_heads, size_t head_dim, size_t page_tokens) {
    KvLayout l{};
    const size_t codes = page_tokens * head_dim * bits / 8, scales = page_tokens * (head_dim / kKvGroup) * 2;
    l.v_off = codes;
    l.ks_off = 2 * codes;
    l.vs_off = 2 * codes + scales;
    l.region = 2 * (codes + scales);
    l.page_bytes = kv_heads * l.region;
    l.page_tokens = (int)page_tokens;
    l.kv_heads = (int)kv_heads;
    l.head_dim = (int)head_dim;
    l.bits = (int)bits;
    return l;
}

struct RopeArgs {
    Heads q, k, q_out, k_out;
    const float *q_weight, *k_weight, *inv_freq;
    const int32_t *positions;
    size_t tokens;
    int head_dim, rot_dim, interleaved;
    float eps, rope_scale;
};
hipError_t launch_qk_norm_rope(const RopeArgs &a, int x_f16, int y_f16, hipStream_t stream);

hipError_t launch_kv_write(uint8_t *pages, size_t page_count, const KvLayout &l, const Heads &k, const Heads &v,
                           int x_f16, size_t tokens, const int64_t *slots, int *bad, hipStream_t stream);
hipError_t launch_kv_read(const uint8_t *pages, size_t page_count, const KvLayout &l, const int64_t *slots,
                          size_t tokens, const Heads &k, const Heads &v, int y_f16, int *bad, hipStream_t stream);

struct CachedArgs {
    Heads q, out;
    const uint8_t *pages;
    size_t page_count, table_stride;
    KvLayout l;
    const int32_t *page_table, *kv_lens;
    int sequences, q_len;
    float scale;
};
// whether the grid and the counts of arrived parts (one word per row tile and sequence, in the
// workspace's exchange) hold the call
bool attention_cached_fits(size_t q_heads, size_t kv_heads, size_t sequences, size_t q_len);
size_t attention_cached_bytes(size_t q_heads, size_t kv_heads, size_t head_dim, size_t sequences, size_t q_len);
hipError_t launch_attention_cached(const CachedArgs &a, void *workspace, hipStream_t stream);

struct PromptArgs {
    Heads q, k, v, out;
    const int32_t *q_starts, *kv_starts;
    int head_dim, sequences, q_tokens, kv_tokens, causal;
    float scale;
};
// 0: the call takes no workspace
size_t attention_prompt_bytes(size_t q_heads, int head_dim, int sequences, int q_tokens, int kv_tokens);
hipError_t launch_attention_prompt(const PromptArgs &a, void *workspace, hipStream_t stream);

}  // namespace exl3k

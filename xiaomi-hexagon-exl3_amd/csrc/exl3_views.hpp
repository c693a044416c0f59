// exl3_views.hpp -- argument checks that the C-ABI's files on rows of heads share (host only).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "exl3_attention.hpp"
#include "exl3_hip.h"

namespace exl3k {

constexpr size_t kMaxHeads = 1024;
constexpr size_t kMaxTokens = (size_t)1 << 30;   // rows of a view: 32-bit row numbers in the kernels
constexpr size_t kMaxSequences = 65536;
constexpr size_t kMaxStride = (size_t)1 << 40;   // elements
constexpr size_t kMaxSpan = (size_t)1 << 48;     // elements from a view's first token (head) to its last: sums of the two
                                                 // and their bytes stay far below 2^64

inline exl3_status from_hip(hipError_t e) { return e == hipSuccess ? EXL3_OK : EXL3_HIP_ERROR; }
inline bool aligned(const void *p, size_t a) { return ((uintptr_t)p % a) == 0; }
inline bool valid_dtype(exl3_dtype t) { return t == EXL3_F32 || t == EXL3_F16; }
inline size_t dtype_size(exl3_dtype t) { return t == EXL3_F16 ? 2 : 4; }

// A head view as the kernels take it.  A view that is written must have disjoint heads:
// its heads lie inside a token's stride or its tokens inside a head's.
inline bool head_view(const exl3_head_view *v, size_t tokens, size_t head_dim, exl3_dtype t, bool written,
                      Heads *out) {
    if (!v || (tokens && !v->data) || !aligned(v->data, dtype_size(t))) return false;
    if (v->heads < 1 || v->heads > kMaxHeads || v->token_stride > kMaxStride || v->head_stride > kMaxStride)
        return false;
    if ((tokens > 1 && v->token_stride > kMaxSpan / (tokens - 1)) ||
        (v->heads > 1 && v->head_stride > kMaxSpan / (v->heads - 1)))
        return false;
    if (written) {
        const bool by_token = (v->heads == 1 || v->head_stride >= head_dim) &&
                              (tokens <= 1 || v->token_stride >= (v->heads - 1) * v->head_stride + head_dim);
        const bool by_head = (tokens <= 1 || v->token_stride >= head_dim) &&
                             (v->heads == 1 || v->head_stride >= (tokens - 1) * v->token_stride + head_dim);
        if (!by_token && !by_head) return false;
    }
    out->data = v->data;
    out->token_stride = v->token_stride;
    out->head_stride = v->head_stride;
    out->heads = (int)v->heads;
    const size_t run = 16 / dtype_size(t);
    out->vec = aligned(v->data, 16) && v->token_stride % run == 0 && v->head_stride % run == 0;
    return true;
}

inline bool same_view(const Heads &a, const Heads &b) {
    return a.data == b.data && a.token_stride == b.token_stride && a.head_stride == b.head_stride;
}

}  // namespace exl3k

// exl3_linear_attention.hpp -- internal interface between the C-ABI of the linear-attention block
// (exl3_linear_attention_api.cpp) and its gfx950 kernels (exl3_rms_norm.hip, exl3_short_conv.hip,
// exl3_delta_{step,prompt}.hip).  Launchers assume validated arguments; they only enqueue work
// and return hipGetLastError().
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "exl3_attention.hpp"

namespace exl3k {

struct NormArgs {
    Heads x, gate, res, res_out, out;  // data null where left out
    const float *weight;
    size_t tokens;
    int width, x_f16, res_f16, y_f16;
    int vec;  // every run of eight elements of each view is 16-byte aligned, and width whole runs
    float eps;
};
hipError_t launch_rms_norm(const NormArgs &a, hipStream_t stream);

// Packed sequences and the states that they start from and leave.
struct Sequences {
    const int32_t *starts;  // null: `tokens / sequences` rows each
    const int32_t *slots_in, *slots_out;
    int sequences, tokens;
    int slots;
};

struct ConvArgs {
    Sequences s;
    const void *x;
    void *y, *states;
    const float *weight, *bias;
    size_t x_stride, y_stride;
    int channels, width, silu;
    int vec;  // eight channels at a time: whole runs of eight, 16-byte aligned
};
hipError_t launch_short_conv(const ConvArgs &a, int x_f16, int y_f16, hipStream_t stream);

struct DeltaArgs {
    Sequences s;
    Heads q, k, v, out;
    const float *g, *beta, *a_log, *dt_bias;
    size_t gate_stride;
    float *states;
    int key_dim, value_dim;
    float scale, eps;  // eps < 0: q and k as they are
};
hipError_t launch_delta_step(const DeltaArgs &a, hipStream_t stream);
// Rows a sequence from which on the chunks take over, and from which on where the sequences, their heads and groups of 16
// columns are kDeltaManyParts or more.  16 heads of 128 x 128: one sequence of 12 rows row by row 11.6 us, of 15 rows
// 13.4 us, of 16 to 24 rows in chunks 15.2 us; 16 sequences of 23 rows 31.4 us row by row, of 24 rows 35.5 us in chunks;
// 64 of 23 rows 96 us, of 24 rows 106 us.
constexpr size_t kDeltaPromptRows = 16, kDeltaPromptRowsOfMany = 24, kDeltaManyParts = 512;
// Packed sequences' lengths are on the device, and a call of few rows a sequence can have a long one among them: from
// kDeltaMixedRows a sequence on, those shorter than kDeltaShortRows go row by row beside the preparation of the others'
// chunks, which takes about as long.  (Five sequences of up to 39 rows, 6 heads of 128 x 256: 18 us, and 23 us where
// short is fewer than 16 rows.  63 single rows and a prompt of 150, 16 heads: 45 us; with a prompt of 60, fewer than two
// rows a sequence, row by row 60 us; 64 sequences of three rows, whose lengths the device alone knows: 39 us, row by row
// 30 us.)
constexpr size_t kDeltaMixedRows = 2, kDeltaShortRows = 8;
// 0: such calls go row by row and take no workspace
size_t delta_prompt_bytes(size_t heads, int key_dim, size_t sequences, size_t tokens);
// Whether this call has chunks: sequences of one known length that is long enough, or packed ones; and a chunk's rows are
// within 32-bit byte offsets of its first
bool delta_prompt_serves(const DeltaArgs &a);
hipError_t launch_delta_prompt(const DeltaArgs &a, void *workspace, hipStream_t stream);

}  // namespace exl3k

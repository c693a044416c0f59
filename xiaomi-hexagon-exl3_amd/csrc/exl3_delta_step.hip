// exl3_delta_step.hip -- the gated delta rule row by row, alone.
#include <limits.h>

#include "exl3_delta_step.hpp"

namespace exl3k {

namespace {

template <int KD>
__global__ __launch_bounds__(64 * kStepWaves) void delta_step_kernel(DeltaArgs a, size_t units, int slices) {
    const size_t unit = (size_t)blockIdx.x * kStepWaves + (threadIdx.x >> 6);
    if (unit < units) delta_step<KD>(a, unit, slices, INT_MAX);
}

}  // namespace

hipError_t launch_delta_step(const DeltaArgs &a, hipStream_t stream) {
    const int slices = (a.value_dim + 15) / 16;
    const size_t units = (size_t)a.s.sequences * a.v.heads * slices;
    const dim3 blocks((unsigned)((units + kStepWaves - 1) / kStepWaves)), threads(64 * kStepWaves);
    if (a.key_dim == 64) delta_step_kernel<64><<<blocks, threads, 0, stream>>>(a, units, slices);
    else delta_step_kernel<128><<<blocks, threads, 0, stream>>>(a, units, slices);
    return hipGetLastError();
}

}  // namespace exl3k

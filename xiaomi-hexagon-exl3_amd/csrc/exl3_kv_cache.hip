// exl3_kv_cache.hip -- the quantised cache: rows of keys and values into their slots and back.
#include "exl3_head_rows.hpp"

namespace exl3k {

namespace {

constexpr int kKvThreads = 256;

__device__ __forceinline__ float group_max(float v) {
    v = fmaxf(v, dpp_xor<1>(v));
    return fmaxf(v, dpp_xor<2>(v));
}

// The scale of a group (fp16 bits) from its largest and smallest element: -ext / 2^(bits-1),
// its magnitude rounded up to 12 - bits significant bits; +0 where that is zero, NaN where
// it is not finite.
template <int BITS>
__device__ __forceinline__ uint16_t group_scale(float top, float low) {
    constexpr uint32_t step = 1u << (BITS - 1);
    const float ext = top > -low ? top : low;
    const uint32_t raw = float_to_half_bits(ext * (-1.0f / step));
    const uint32_t s = (raw + (step - 1)) & ~(step - 1);
    if ((raw & 0x7fffu) >= 0x7c00u || (s & 0x7fffu) >= 0x7c00u) return 0x7e00u;
    return (s & 0x7fffu) ? (uint16_t)s : (uint16_t)0;
}

// One lane group of D / 8 lanes quantises one head's key or value row of one token.
template <int D, int BITS, int XF16>
__global__ __launch_bounds__(kKvThreads) void kv_write_kernel(uint8_t *__restrict__ pages, size_t slot_count,
                                                              KvLayout lay, Heads k, Heads v, size_t tokens,
                                                              const int64_t *__restrict__ slots, int *bad) {
    constexpr int VL = D / 8;
    const int lane = threadIdx.x & 63, l = threadIdx.x & (VL - 1);
    const size_t rows = 2 * (size_t)k.heads, units = tokens * rows;
    for (size_t unit = (size_t)blockIdx.x * (kKvThreads / VL) + threadIdx.x / VL; unit < units;
         unit += (size_t)gridDim.x * (kKvThreads / VL)) {  // whole lane groups
        const size_t token = unit / rows;
        const int row = (int)(unit - token * rows);
        const int is_v = row >= k.heads, head = is_v ? row - k.heads : row;
        const int64_t slot = slots[token];
        if (slot < 0 || (size_t)slot >= slot_count) {
            if (slot >= 0 && bad && row == 0 && l == 0) *bad = 1;
            continue;
        }
        const Heads &in = is_v ? v : k;
        float x[8];
        load_run8<XF16>(in.data, token * in.token_stride + head * in.head_stride + 8 * l, in.vec, x);
        h32_run8(x, lane);
        float top = x[0], low = x[0];
    #pragma unroll
        for (int e = 1; e < 8; ++e) {
            top = fmaxf(top, x[e]);
            low = fminf(low, x[e]);
        }
        top = group_max(top);
        low = -group_max(-low);
        const uint16_t sb = group_scale<BITS>(top, low);
        const float s = half_bits_to_float(sb);
        const float r = s == 0.f ? 0.f : 1.0f / s;
        constexpr int H = 1 << (BITS - 1);
        uint32_t code[8];
    #pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float c = fminf(fmaxf(__builtin_rintf(x[e] * r), (float)-H), (float)(H - 1));
            code[e] = (uint32_t)((int)c + H);
        }
        const int p = lay.page_tokens;
        const size_t page = (size_t)slot / p;
        const int at = (int)((size_t)slot - page * p);
        uint8_t *base = pages + page * lay.page_bytes + (size_t)head * lay.region;
        uint32_t w[BITS / 4];
        if constexpr (BITS == 4) {
            w[0] = 0;
    #pragma unroll
            for (int e = 0; e < 8; ++e) w[0] |= code[e] << (4 * e);
        } else {
            w[0] = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
            w[1] = code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24;
        }
        constexpr int RUN = D * BITS / 8;     // bytes of a row
        constexpr int PART = D * BITS / 128;  // bytes of one of a value row's 16 slices
        if (!is_v) {
            uint32_t *o = (uint32_t *)(base + (size_t)at * RUN + l * BITS);
    #pragma unroll
            for (int i = 0; i < BITS / 4; ++i) o[i] = w[i];
            if ((l & 3) == 0)
                *(uint16_t *)(base + lay.ks_off + (size_t)at * (D / kKvGroup * 2) + (l >> 2) * 2) = sb;
        } else {
            uint8_t *blk = base + lay.v_off + (size_t)(at >> 2) * (4 * RUN) + (at & 3) * PART;
            if constexpr (PART <= BITS) {  // D <= 128: a lane's eight elements are BITS / PART whole slices
    #pragma unroll
                for (int i = 0; i < BITS / PART; ++i) {
                    uint8_t *o = blk + (size_t)(l * (BITS / PART) + i) * (4 * PART);
                    if constexpr (PART == 2) *(uint16_t *)o = (uint16_t)(w[0] >> (16 * i));
                    else if constexpr (PART == 4) *(uint32_t *)o = w[i];
                    else *(u2 *)o = (u2){w[0], w[BITS / 4 - 1]};
                }
            } else {  // D = 256: two lanes fill one slice
                uint8_t *o = blk + (size_t)(l >> 1) * (4 * PART) + (l & 1) * BITS;
    #pragma unroll
                for (int i = 0; i < BITS / 4; ++i) ((uint32_t *)o)[i] = w[i];
            }
            if ((l & 3) == 0)
                *(uint16_t *)(base + lay.vs_off + (size_t)(at >> 2) * (D / kKvGroup * 8) + (l >> 2) * 8 + (at & 3) * 2) = sb;
        }
    }
}

template <int D, int BITS, int YF16>
__global__ __launch_bounds__(kKvThreads) void kv_read_kernel(const uint8_t *__restrict__ pages, size_t slot_count,
                                                             KvLayout lay, const int64_t *__restrict__ slots,
                                                             size_t tokens, Heads k, Heads v, int *bad) {
    constexpr int VL = D / 8, RUN = D * BITS / 8, PART = D * BITS / 128;
    const int lane = threadIdx.x & 63, l = threadIdx.x & (VL - 1);
    const size_t rows = 2 * (size_t)k.heads, units = tokens * rows;
    for (size_t unit = (size_t)blockIdx.x * (kKvThreads / VL) + threadIdx.x / VL; unit < units;
         unit += (size_t)gridDim.x * (kKvThreads / VL)) {  // whole lane groups
        const size_t token = unit / rows;
        const int row = (int)(unit - token * rows);
        const int is_v = row >= k.heads, head = is_v ? row - k.heads : row;
        const int64_t slot = slots[token];
        float x[8];
        if (slot < 0 || (size_t)slot >= slot_count) {
            if (bad && row == 0 && l == 0) *bad = 1;
    #pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __builtin_nanf("");
        } else {
            const int p = lay.page_tokens;
            const size_t page = (size_t)slot / p;
            const int at = (int)((size_t)slot - page * p);
            const uint8_t *base = pages + page * lay.page_bytes + (size_t)head * lay.region;
            uint32_t w[BITS / 4];
            float s;
            if (!is_v) {
                const uint32_t *o = (const uint32_t *)(base + (size_t)at * RUN + l * BITS);
    #pragma unroll
                for (int i = 0; i < BITS / 4; ++i) w[i] = o[i];
                s = half_bits_to_float(*(const uint16_t *)(base + lay.ks_off + (size_t)at * (D / kKvGroup * 2) + (l >> 2) * 2));
            } else {
                const uint8_t *blk = base + lay.v_off + (size_t)(at >> 2) * (4 * RUN) + (at & 3) * PART;
                if constexpr (PART <= BITS) {
                    w[0] = 0;
    #pragma unroll
                    for (int i = 0; i < BITS / PART; ++i) {
                        const uint8_t *o = blk + (size_t)(l * (BITS / PART) + i) * (4 * PART);
                        if constexpr (PART == 2) w[0] |= (uint32_t)*(const uint16_t *)o << (16 * i);
                        else if constexpr (PART == 4) w[i] = *(const uint32_t *)o;
                        else {
                            w[0] = ((const uint32_t *)o)[0];
                            w[BITS / 4 - 1] = ((const uint32_t *)o)[1];
                        }
                    }
                } else {
                    const uint8_t *o = blk + (size_t)(l >> 1) * (4 * PART) + (l & 1) * BITS;
    #pragma unroll
                    for (int i = 0; i < BITS / 4; ++i) w[i] = ((const uint32_t *)o)[i];
                }
                s = half_bits_to_float(
                    *(const uint16_t *)(base + lay.vs_off + (size_t)(at >> 2) * (D / kKvGroup * 8) + (l >> 2) * 8 + (at & 3) * 2));
            }
            constexpr int H = 1 << (BITS - 1), PER = 32 / BITS;
    #pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] = (float)((int)((w[e / PER] >> (e % PER * BITS)) & ((1u << BITS) - 1)) - H) * s;
            h32_run8(x, lane);
        }
        const Heads &out = is_v ? v : k;
        store_run8<YF16>(out.data, token * out.token_stride + head * out.head_stride + 8 * l, out.vec, x);
    }
}

template <int D, int BITS>
hipError_t write_db(uint8_t *pages, size_t slots_n, const KvLayout &l, const Heads &k, const Heads &v, int x_f16,
                    size_t tokens, const int64_t *slots, int *bad, hipStream_t stream) {
    const unsigned blocks = row_blocks(tokens * 2 * k.heads, kKvThreads / (D / 8));
    if (x_f16)
        kv_write_kernel<D, BITS, 1><<<dim3(blocks), dim3(kKvThreads), 0, stream>>>(pages, slots_n, l, k, v, tokens, slots, bad);
    else
        kv_write_kernel<D, BITS, 0><<<dim3(blocks), dim3(kKvThreads), 0, stream>>>(pages, slots_n, l, k, v, tokens, slots, bad);
    return hipGetLastError();
}
template <int D, int BITS>
hipError_t read_db(const uint8_t *pages, size_t slots_n, const KvLayout &l, const int64_t *slots, size_t tokens,
                   const Heads &k, const Heads &v, int y_f16, int *bad, hipStream_t stream) {
    const unsigned blocks = row_blocks(tokens * 2 * k.heads, kKvThreads / (D / 8));
    if (y_f16)
        kv_read_kernel<D, BITS, 1><<<dim3(blocks), dim3(kKvThreads), 0, stream>>>(pages, slots_n, l, slots, tokens, k, v, bad);
    else
        kv_read_kernel<D, BITS, 0><<<dim3(blocks), dim3(kKvThreads), 0, stream>>>(pages, slots_n, l, slots, tokens, k, v, bad);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_write(uint8_t *pages, size_t page_count, const KvLayout &l, const Heads &k, const Heads &v,
                           int x_f16, size_t tokens, const int64_t *slots, int *bad, hipStream_t stream) {
    const size_t n = page_count * l.page_tokens;
    switch (l.head_dim * 16 + l.bits) {
    case 64 * 16 + 4: return write_db<64, 4>(pages, n, l, k, v, x_f16, tokens, slots, bad, stream);
    case 64 * 16 + 8: return write_db<64, 8>(pages, n, l, k, v, x_f16, tokens, slots, bad, stream);
    case 128 * 16 + 4: return write_db<128, 4>(pages, n, l, k, v, x_f16, tokens, slots, bad, stream);
    case 128 * 16 + 8: return write_db<128, 8>(pages, n, l, k, v, x_f16, tokens, slots, bad, stream);
    case 256 * 16 + 4: return write_db<256, 4>(pages, n, l, k, v, x_f16, tokens, slots, bad, stream);
    default: return write_db<256, 8>(pages, n, l, k, v, x_f16, tokens, slots, bad, stream);
    }
}

hipError_t launch_kv_read(const uint8_t *pages, size_t page_count, const KvLayout &l, const int64_t *slots,
                          size_t tokens, const Heads &k, const Heads &v, int y_f16, int *bad, hipStream_t stream) {
    const size_t n = page_count * l.page_tokens;
    switch (l.head_dim * 16 + l.bits) {
    case 64 * 16 + 4: return read_db<64, 4>(pages, n, l, slots, tokens, k, v, y_f16, bad, stream);
    case 64 * 16 + 8: return read_db<64, 8>(pages, n, l, slots, tokens, k, v, y_f16, bad, stream);
    case 128 * 16 + 4: return read_db<128, 4>(pages, n, l, slots, tokens, k, v, y_f16, bad, stream);
    case 128 * 16 + 8: return read_db<128, 8>(pages, n, l, slots, tokens, k, v, y_f16, bad, stream);
    case 256 * 16 + 4: return read_db<256, 4>(pages, n, l, slots, tokens, k, v, y_f16, bad, stream);
    default: return read_db<256, 8>(pages, n, l, slots, tokens, k, v, y_f16, bad, stream);
    }
}

}  // namespace exl3k

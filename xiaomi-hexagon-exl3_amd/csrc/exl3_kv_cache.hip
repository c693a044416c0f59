// exl3_kv_cache.hip -- the quantised cache: rows of keys and values into their slots and back.
//
// A row is rotated by H32 per 32 elements, which spreads an outlier over its group, and each group is kept as codes
// times one fp16 scale.  Both ways are one pass, bound by the rows' bytes: 16,384 tokens, 8 heads of 128 in fp16
// at 4 bits: written in 22.8 us (3.8 TB/s with the cache's), read in 18.7 (4.6); eight tokens: 2.7 and 2.6 us.
#include "exl3_head_rows.hpp"

namespace exl3k {

namespace {

constexpr int kKvThreads = 256;
constexpr size_t kKvGroups = 2048;  // workgroups that fill the chip: 256 CUs, eight each

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

// A place in the cache, or none.
struct Place {
    size_t page;  // byte offset
    int at;       // token of the page
    bool in;
};
__device__ __forceinline__ Place place_of(int64_t slot, size_t slot_count, const KvLayout &lay) {
    Place p;
    p.in = slot >= 0 && (size_t)slot < slot_count;
    const uint32_t s = p.in ? (uint32_t)(slot / 16) : 0;  // pages are whole pieces of 16 tokens, at most 2^44 of them
    const uint64_t pieces = p.in ? (uint64_t)slot / 16 : 0;
    const uint32_t per = (uint32_t)lay.page_tokens / 16;
    const uint64_t page = pieces <= 0xffffffffu ? s / per : pieces / per;
    p.page = page * lay.page_bytes;
    p.at = (int)(pieces - page * per) * 16 + (int)(slot & 15);
    return p;
}

// D / 8 lanes hold one head's key or value row of one token, eight elements each, and walk the
// heads; neighbouring lanes' tokens are neighbours, so what a run of slots writes (a value block's four
// tokens, the scales) comes from one wave.  Bound by the rows' bytes: the next row is asked for before
// this one is worked on.
template <int D, int BITS, int XF16>
__global__ __launch_bounds__(kKvThreads) void kv_write_kernel(uint8_t *__restrict__ pages, size_t slot_count,
                                                              KvLayout lay, Heads k, Heads v, size_t tokens,
                                                              const int64_t *__restrict__ slots, int *bad, int slices) {
    constexpr int VL = D / 8, kTokens = kKvThreads / VL;
    constexpr int RUN = D * BITS / 8;     // bytes of a row
    constexpr int PART = D * BITS / 128;  // bytes of one of a value row's 16 slices
    constexpr int H = 1 << (BITS - 1), G = D / kKvGroup;
    const int lane = threadIdx.x & 63, l = threadIdx.x & (VL - 1), slice = blockIdx.x % slices, rows = 2 * k.heads;
    for (size_t token = (size_t)(blockIdx.x / slices) * kTokens + threadIdx.x / VL; token < tokens;
         token += (size_t)(gridDim.x / slices) * kTokens) {  // whole lane groups
        auto fetch = [&](int row, float (&x)[8]) {
            const Heads &in = row >= k.heads ? v : k;
            const int head = row >= k.heads ? row - k.heads : row;
            load_run8<XF16>(in.data, token * in.token_stride + head * in.head_stride + 8 * l, in.vec, x);
        };
        float next[8];
        fetch(slice, next);
        const int64_t slot = slots[token];
        const Place to = place_of(slot, slot_count, lay);
        if (!to.in) {
            if (slot >= 0 && bad && slice == 0 && l == 0) *bad = 1;
            continue;
        }
        for (int row = slice; row < rows; row += slices) {
            const bool is_v = row >= k.heads;
            const int head = is_v ? row - k.heads : row;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = next[e];
            if (row + slices < rows) fetch(row + slices, next);
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
            // code + H in the low bits: adding 1.5 * 2^23 rounds to the nearest whole number (ties to even), and
            // the sum's upper bits, the same for every element, fall out of the words by a last difference.  The
            // lowest code needs no bound: only the extreme gets there, from at most 2^-11 beyond.
            uint32_t w[BITS / 4] = {};
            constexpr int PER = 32 / BITS;
#pragma unroll
            for (int e = 7; e >= 0; --e) {
                const float c = fminf(x[e] * r, (float)(H - 1)) + (12582912.f + H);
                w[e / PER] = (w[e / PER] << BITS) + __float_as_uint(c);
            }
            uint32_t upper = 0;
            for (int e = 0; e < PER; ++e) upper = (upper << BITS) + 0x4b400000u;
#pragma unroll
            for (int i = 0; i < BITS / 4; ++i) w[i] -= upper;
            uint8_t *base = pages + to.page + (size_t)head * lay.region;
            if (!is_v) {
                uint32_t *o = (uint32_t *)(base + (size_t)to.at * RUN + l * BITS);
                if constexpr (BITS == 4) *o = w[0];
                else *(u2 *)o = (u2){w[0], w[1]};
                if ((l & 3) == 0) *(uint16_t *)(base + lay.ks_off + (size_t)to.at * (2 * G) + (l >> 2) * 2) = sb;
            } else {
                uint8_t *blk = base + lay.v_off + (size_t)(to.at >> 2) * (4 * RUN) + (to.at & 3) * PART;
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
                    if constexpr (BITS == 4) *(uint32_t *)o = w[0];
                    else *(u2 *)o = (u2){w[0], w[1]};
                }
                if ((l & 3) == 0)
                    *(uint16_t *)(base + lay.vs_off + (size_t)(to.at >> 2) * (8 * G) + (l >> 2) * 8 + (to.at & 3) * 2) = sb;
            }
        }
    }
}

template <int D, int BITS, int YF16>
__global__ __launch_bounds__(kKvThreads) void kv_read_kernel(const uint8_t *__restrict__ pages, size_t slot_count,
                                                             KvLayout lay, const int64_t *__restrict__ slots,
                                                             size_t tokens, Heads k, Heads v, int *bad, int slices) {
    constexpr int VL = D / 8, RUN = D * BITS / 8, PART = D * BITS / 128, kTokens = kKvThreads / VL;
    constexpr int H = 1 << (BITS - 1), PER = 32 / BITS, G = D / kKvGroup;
    const int lane = threadIdx.x & 63, l = threadIdx.x & (VL - 1), slice = blockIdx.x % slices, rows = 2 * k.heads;
    for (size_t token = (size_t)(blockIdx.x / slices) * kTokens + threadIdx.x / VL; token < tokens;
         token += (size_t)(gridDim.x / slices) * kTokens) {  // whole lane groups
        const int64_t slot = slots[token];
        const Place from = place_of(slot, slot_count, lay);
        if (!from.in && bad && slice == 0 && l == 0) *bad = 1;
        struct Codes {
            uint32_t w[BITS / 4];
            uint16_t s;
        };
        auto fetch = [&](int row, Codes &c) {  // a place outside the cache: zeros under a NaN scale
            const bool is_v = row >= k.heads;
            const int head = is_v ? row - k.heads : row;
            const uint8_t *base = pages + from.page + (size_t)head * lay.region;
#pragma unroll
            for (int i = 0; i < BITS / 4; ++i) c.w[i] = 0;
            c.s = 0x7e00;
            if (!from.in) return;
            if (!is_v) {
                const uint32_t *o = (const uint32_t *)(base + (size_t)from.at * RUN + l * BITS);
                if constexpr (BITS == 4) c.w[0] = *o;
                else {
                    const u2 t = *(const u2 *)o;
                    c.w[0] = t.x;
                    c.w[1] = t.y;
                }
                c.s = *(const uint16_t *)(base + lay.ks_off + (size_t)from.at * (2 * G) + (l >> 2) * 2);
            } else {
                const uint8_t *blk = base + lay.v_off + (size_t)(from.at >> 2) * (4 * RUN) + (from.at & 3) * PART;
                if constexpr (PART <= BITS) {
#pragma unroll
                    for (int i = 0; i < BITS / PART; ++i) {
                        const uint8_t *o = blk + (size_t)(l * (BITS / PART) + i) * (4 * PART);
                        if constexpr (PART == 2) c.w[0] |= (uint32_t)*(const uint16_t *)o << (16 * i);
                        else if constexpr (PART == 4) c.w[i] = *(const uint32_t *)o;
                        else {
                            const u2 t = *(const u2 *)o;
                            c.w[0] = t.x;
                            c.w[BITS / 4 - 1] = t.y;
                        }
                    }
                } else {
                    const uint8_t *o = blk + (size_t)(l >> 1) * (4 * PART) + (l & 1) * BITS;
#pragma unroll
                    for (int i = 0; i < BITS / 4; ++i) c.w[i] = ((const uint32_t *)o)[i];
                }
                c.s = *(const uint16_t *)(base + lay.vs_off + (size_t)(from.at >> 2) * (8 * G) + (l >> 2) * 8 + (from.at & 3) * 2);
            }
        };
        Codes next;
        fetch(slice, next);
        for (int row = slice; row < rows; row += slices) {
            const bool is_v = row >= k.heads;
            const int head = is_v ? row - k.heads : row;
            const Codes c = next;
            if (row + slices < rows) fetch(row + slices, next);
            const float s = half_bits_to_float(c.s);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                x[e] = (float)((int)((c.w[e / PER] >> (e % PER * BITS)) & ((1u << BITS) - 1)) - H) * s;
            h32_run8(x, lane);
            const Heads &out = is_v ? v : k;
            store_run8<YF16>(out.data, token * out.token_stride + head * out.head_stride + 8 * l, out.vec, x);
        }
    }
}

template <int D, int BITS>
hipError_t write_db(uint8_t *pages, size_t slots_n, const KvLayout &l, const Heads &k, const Heads &v, int x_f16,
                    size_t tokens, const int64_t *slots, int *bad, hipStream_t stream) {
    const RowGrid g = row_grid(tokens, kKvThreads / (D / 8), 2 * k.heads, kKvGroups);
    if (x_f16)
        kv_write_kernel<D, BITS, 1><<<g.blocks, kKvThreads, 0, stream>>>(pages, slots_n, l, k, v, tokens, slots, bad, g.slices);
    else
        kv_write_kernel<D, BITS, 0><<<g.blocks, kKvThreads, 0, stream>>>(pages, slots_n, l, k, v, tokens, slots, bad, g.slices);
    return hipGetLastError();
}
template <int D, int BITS>
hipError_t read_db(const uint8_t *pages, size_t slots_n, const KvLayout &l, const int64_t *slots, size_t tokens,
                   const Heads &k, const Heads &v, int y_f16, int *bad, hipStream_t stream) {
    const RowGrid g = row_grid(tokens, kKvThreads / (D / 8), 2 * k.heads, kKvGroups);
    if (y_f16)
        kv_read_kernel<D, BITS, 1><<<g.blocks, kKvThreads, 0, stream>>>(pages, slots_n, l, slots, tokens, k, v, bad, g.slices);
    else
        kv_read_kernel<D, BITS, 0><<<g.blocks, kKvThreads, 0, stream>>>(pages, slots_n, l, slots, tokens, k, v, bad, g.slices);
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

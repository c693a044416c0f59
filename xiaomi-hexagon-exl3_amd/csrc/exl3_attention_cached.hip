// exl3_attention_cached.hip -- attention of each sequence's last tokens over the quantised cache.
//
// One pass over the cached tokens: 16 query rows (the q heads of one kv head times the new
// tokens) meet every key, with the running maximum and sum of the softmax.  Bound by the
// cache's bytes: a token of one kv head is D * bits / 4 + D / 8 bytes and 2 * 16 * 2 D
// multiply-adds on the matrix cores.  Workgroups share a long sequence; the last of them to end joins their parts, or
// a second kernel does.
//
// A wave takes 32 tokens at a time and computes S^T = K Q^T and O^T = V^T P^T with
// mfma_f32_16x16x32_f16.  The layout of the page makes each operand one or two wide loads and a
// few VALU operations per eight codes, with no exchange between lanes and no LDS:
//   K: lane (m = lane % 16, g = lane / 16) holds a quarter of key m's row, so 16 keys are one
//      contiguous run; the k index of MFMA j is element g D / 4 + 8 j + e, of the queries too.
//   S^T leaves lane (row, g) with keys 4 g .. 4 g + 3 of each 16: as the B operand of the second
//      product these are its k indices 8 g + (0 .. 3) and, from the second 16 keys, 8 g + (4 .. 7).
//   V: a lane's block of four tokens holds those four keys for its slice of D / 16 elements;
//      the A operand of O^T tile t is element t of the slice: row m of the tile is element
//      m D / 16 + t of the head.
// Dequantising adds no rounding and leaves no value out of fp16's range (Masks).  The queries are
// rotated by H32 like the cached rows and kept as an fp16 pair (high and low part: two
// MFMAs, which the VALU work hides; a row that the rotation could take beyond fp16's range is kept as an eighth, with
// eight times its factor in the exponent); the result is rotated back at the end.
// 16 sequences of 32,768 tokens, 32 / 8 heads of 128 at 4 bits (604 MB): 117 to 122 us, 5.0 to 5.2 TB/s, the rate of a
// large copy, with the VALU at work 62 % of the time; of 20,000 at 8 bits: 124 us, 5.6 TB/s; 1,000 tokens, 8 / 2
// heads of 256: 13.2 us, a launch and four dependent round trips.
#include "exl3_head_rows.hpp"

namespace exl3k {

namespace {

constexpr int kTile = 32;                          // tokens of a wave's step
constexpr int kRows = 16;                          // query rows of a workgroup
// Waves of a workgroup: as many as the registers of a CU hold (two waves per SIMD, one at head
// dimension 256), so that a part to be joined covers as many tokens as can be.
constexpr int cached_waves(int d) { return d == 256 ? 4 : 8; }
constexpr int kCachedGroups = 256;                 // workgroups: one per CU
// Units of a sequence up to which each has a workgroup (1,000 tokens, 4 rows of 256: 13.4 us against 14.5
// shared out; with 576 workgroups, most of them without tokens, 17.0 against 13.6).
constexpr int kDirectUnits = 8;
constexpr float kStart = -1e30f;                   // running maximum before the first key
constexpr float kSlack = 8.f;                      // scores may pass the running maximum by 2^8
constexpr float kLog2e = 1.4426950408889634f;
// H32 makes an element at most sqrt(32) times a row's largest: up to this fp16 value the rotated row is within
// 65,504.  A row beyond it is kept as an eighth (46,319 at most), the other rows as they are.
constexpr float kFullQuery = 11576.f;

// The work in units of a tile for every wave.  Either (few units: `direct`) a workgroup for each unit of
// each sequence that the page table has room for, which knows its place without the lengths, so that
// lengths, page table and queries come in one round trip, not three; a unit's part of sequence s is partial
// s * direct + unit.  Or the tokens of all sequences are one row of units, which the workers of a kv head
// share evenly: worker w of n has units [w U / n, (w + 1) U / n), and its part of sequence s is partial
// w + s (one of them grows at each step).
template <int UNIT>
struct Share {
    const int32_t *lens;
    long most;  // tokens that the page table can name
    int sequences;
    __device__ __forceinline__ int len(int s) const {
        const int n = lens[s];
        return n < 0 ? 0 : (n > most ? (int)most : n);
    }
    __device__ __forceinline__ int units(int s) const { return s < sequences ? (len(s) + UNIT - 1) / UNIT : 0; }
};
// over the first n lanes, n > 0 (the others hold zero)
__device__ __forceinline__ int wave_scan(int v, int lane, int n) {  // inclusive
    for (int d = 1; d < min(n, 64); d <<= 1) {
        const int o = __shfl_up(v, d);
        v += lane >= d ? o : 0;
    }
    return v;
}
// all sequences' units, and those of the longest
template <typename S>
__device__ __forceinline__ long total_units(const S &sh, int lane, int &longest) {
    long all = 0;
    longest = 0;
    for (int s0 = 0; s0 < sh.sequences; s0 += 64) {
        const int n = min(sh.sequences - s0, 64);
        int units = sh.units(s0 + lane);
        all += __builtin_amdgcn_readlane(wave_scan(units, lane, n), n - 1);
        for (int d = 1; d < n; d <<= 1) units = max(units, __shfl_xor(units, d));
        longest = max(longest, __builtin_amdgcn_readfirstlane(units));
    }
    return all;
}
// Units of a worker: t units take t a, and the last worker of a sequence of u units then joins u / t
// parts of `size` elements, b size each, one round trip for eight; the sum is least at t = sqrt(u size b / a).
// b / a = 1 / 8192 is measured: 16,000 tokens, 4 rows of 256 (125 units): t = 1, 2, 4, 8 take 50.9, 33.9, 27.7,
// 30.1 us; 4,000 tokens: 21.9, 19.1, 20.3, 26.7; 16,000 tokens, 4 rows of 64 (63 units): 13.3, 13.0, 14.8, 19.2.
__device__ __forceinline__ int units_each(int longest, int size) {
    return max(1, (int)(__builtin_sqrtf((float)longest * (float)size * (1.f / 8192.f)) + 0.4f));
}
// the sequence that holds unit u (u < the total), and its first unit
template <typename S>
__device__ __forceinline__ int find_unit(const S &sh, long u, int lane, long &first) {
    long before = 0;
    for (int s0 = 0;; s0 += 64) {
        const int n = sh.units(s0 + lane);
        const int end = wave_scan(n, lane, sh.sequences - s0);
        const unsigned long long hit = __ballot(u < before + end);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            first = before + __builtin_amdgcn_readlane(end - n, l);
            return s0 + l;
        }
        before += __builtin_amdgcn_readlane(end, 63);
    }
}

// a b / c for a <= c: 32-bit arithmetic where it holds (a 64-bit division is about 150 instructions)
__device__ __forceinline__ long mul_div(long a, long b, long c) {
    if (b * c <= 0xffffffffl) return (uint32_t)(a * b) / (uint32_t)c;
    return a * b / c;
}

template <int N>
__device__ __forceinline__ void load_words(const uint8_t *p, uint32_t (&w)[N]) {
    if constexpr (N == 2) {
        const u2 t = *(const u2 *)p;
        w[0] = t.x;
        w[1] = t.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const u4 t = ((const u4 *)p)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[4 * i + e] = t[e];
        }
    }
}

// Codes become fp16 numbers code / 2^(BITS - 1), -1 to just below 1, by or-ing them into the last bits of a number
// whose spacing is that (128 at 4 bits, 8 at 8) and taking it off again.  Times a scale of 12 - BITS significant bits
// that is exact to the last subnormal (whole multiples of 2^-24) and within fp16's range for every finite scale
// (65,280 at most), where code * scale is not: 32 equal elements of 12,000 rotate to 67,882.  The power of two is in the
// exponent's factor and in the last division.
// The masks and that number are in registers: a v_and_or_b32 takes no literals, so with constants each is a
// v_and and a v_or.
template <int BITS>
struct Masks {
    uint32_t low, high, base;  // scalar, scalar, vector
    __device__ __forceinline__ Masks() : low(0x000f000fu), high(0x00f000f0u), base(BITS == 4 ? 0x58005800u : 0x48004800u) {
        asm volatile("" : "+s"(low), "+s"(high), "+v"(base));
    }
};
// two 4-bit codes in the halves' bits 0..3, or 4..7: 128 + c / 8 and 128 + 2 c
__device__ __forceinline__ h2 low_codes(uint32_t w, const Masks<4> &k) {
    return bitcast<h2>((w & k.low) | k.base) + (h2){(_Float16)-129.f, (_Float16)-129.f};
}
__device__ __forceinline__ h2 high_codes(uint32_t w, const Masks<4> &k) {
    return __builtin_elementwise_fma(bitcast<h2>((w & k.high) | k.base), (h2){(_Float16)0.0625f, (_Float16)0.0625f},
                                     (h2){(_Float16)-9.f, (_Float16)-9.f});
}
__device__ __forceinline__ h2 byte_codes(uint32_t w, const Masks<8> &k) {  // 8 bits: 8 + c / 128
    return bitcast<h2>(w | k.base) + (h2){(_Float16)-9.f, (_Float16)-9.f};
}

template <int D, int BITS>
struct Cached {
    static constexpr int RUN = D * BITS / 8;   // bytes of a row's codes
    static constexpr int NW = RUN / 16;        // words of a lane's share of 16 keys, or of 4 tokens' slices
    static constexpr int G = D / kKvGroup;     // scale groups of a row
    static constexpr int NJ = D / 32;          // MFMAs over the elements
    static constexpr int NT = D / 16;          // O^T tiles

    struct Half {  // one lane's part of 16 tokens
        uint32_t k[NW], v[NW], ks;
        u2 vs;
    };

    // A lane's places in 16 tokens, the same for all of them: the rest of an address is scalar.
    struct Lane {
        uint32_t k, v, ks, vs;
    };
    static __device__ __forceinline__ Lane lane_of(int m, int g) {
        return {(uint32_t)(m * RUN + g * (RUN / 4)), (uint32_t)(g * (4 * RUN) + m * (RUN / 4)),
                (uint32_t)(m * (2 * G) + (G == 8 ? 4 * g : 2 * (G == 4 ? g : g >> 1))),
                (uint32_t)(g * (8 * G) + 8 * (m * G / 16))};
    }
    // base: the head's region of the page; off: the first token's place in it (a multiple of 16), both scalar
    static __device__ __forceinline__ void load(const uint8_t *base, uint32_t off, const KvLayout &l, const Lane &at, Half &h) {
        load_words<NW>(base + off * (uint32_t)RUN + at.k, h.k);
        load_words<NW>(base + l.v_off + off * (uint32_t)RUN + at.v, h.v);
        const uint8_t *ks = base + l.ks_off + off * (uint32_t)(2 * G) + at.ks;
        if constexpr (G == 8) h.ks = *(const uint32_t *)ks;
        else h.ks = *(const uint16_t *)ks;
        h.vs = *(const u2 *)(base + l.vs_off + off * (uint32_t)(2 * G) + at.vs);
    }

    // Fragment j of a lane's key: elements 8 j .. 8 j + 7 of its quarter row, in the order that
    // q_order undoes.
    static __device__ __forceinline__ h8 key(const Half &h, int j, const Masks<BITS> &c) {
        const uint32_t sw = G == 8 ? (j < 4 ? h.ks & 0xffffu : h.ks >> 16) : h.ks;
        const _Float16 s = bitcast<_Float16>((uint16_t)sw);
        const h2 s2 = {s, s};
        h2 p[4];
        if constexpr (BITS == 4) {
            const uint32_t w = h.k[j], w8 = w >> 8;
            p[0] = low_codes(w, c);
            p[1] = high_codes(w, c);
            p[2] = low_codes(w8, c);
            p[3] = high_codes(w8, c);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                p[i] = byte_codes(__builtin_amdgcn_perm(0u, h.k[2 * j + i / 2], i & 1 ? 0x0c030c02u : 0x0c010c00u), c);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = p[i] * s2;
        return (h8){p[0][0], p[0][1], p[1][0], p[1][1], p[2][0], p[2][1], p[3][0], p[3][1]};
    }
    // eight query elements in natural order, in that order
    static __device__ __forceinline__ h8 q_order(h8 v) {
        if constexpr (BITS == 4) return (h8){v[0], v[4], v[1], v[5], v[2], v[6], v[3], v[7]};
        else return v;
    }

    // element t of the lane's slice for its four tokens (as two pairs)
    static __device__ __forceinline__ void value(const Half &h, int t, h2 &a, h2 &b, const Masks<BITS> &c) {
        const h2 s01 = bitcast<h2>(h.vs.x), s23 = bitcast<h2>(h.vs.y);
        if constexpr (D == 64 && BITS == 4) {  // 2-byte slices: a word holds two tokens
            const uint32_t x = t < 2 ? h.v[0] : h.v[0] >> 8, y = t < 2 ? h.v[1] : h.v[1] >> 8;
            a = (t & 1) ? high_codes(x, c) : low_codes(x, c);
            b = (t & 1) ? high_codes(y, c) : low_codes(y, c);
        } else {
            constexpr int PW = NW / 4;  // words of a token's slice
            const int byte = BITS == 4 ? (t / 2) % 4 : t % 4, word = BITS == 4 ? t / 8 : t / 4;
            const uint32_t sel = 0x0c000c00u + (uint32_t)(byte + ((byte + 4) << 16));
            const uint32_t x = __builtin_amdgcn_perm(h.v[PW + word], h.v[word], sel);
            const uint32_t y = __builtin_amdgcn_perm(h.v[3 * PW + word], h.v[2 * PW + word], sel);
            if constexpr (BITS == 4) {
                a = (t & 1) ? high_codes(x, c) : low_codes(x, c);
                b = (t & 1) ? high_codes(y, c) : low_codes(y, c);
            } else {
                a = byte_codes(x, c);
                b = byte_codes(y, c);
            }
        }
        a = a * s01;
        b = b * s23;
    }
};

__device__ __forceinline__ float over_groups_max(float v) {  // over lanes l ^ 16, l ^ 32
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = fmaxf(__int_as_float(a[0]), __int_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return fmaxf(__int_as_float(b[0]), __int_as_float(b[1]));
}
__device__ __forceinline__ float over_groups_sum(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = __int_as_float(a[0]) + __int_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return __int_as_float(b[0]) + __int_as_float(b[1]);
}

// Partials of one (kv head, row tile): sums [slot][rows][D], then (maximum, sum) [slot][rows], rows the
// real rows of the tile; every tile has room for those of the first, in whole 256 bytes (the join reads 16 at a time).  They cross XCDs, each with its own
// L2, so they are stored and loaded as relaxed agent-scope atomics (coherent at device scope, no cache maintenance; a release fence writes
// back a whole L2).
struct Parts {
    unsigned long long *sums, *stats;  // pairs of binary32
};
__host__ __device__ constexpr size_t part_words(size_t d, size_t rows, size_t slots) {
    return (slots * rows * (d / 2 + 1) + 31) / 32 * 32;
}
__device__ __forceinline__ Parts parts_of(void *ws, int d, int rows, size_t slots, size_t y) {
    Parts p;
    p.sums = (unsigned long long *)ws + y * part_words(d, rows, slots);
    p.stats = p.sums + slots * (size_t)(rows * (d / 2));
    return p;
}
__device__ __forceinline__ void put_pair(unsigned long long *p, float a, float b) {
    __hip_atomic_store(p, (unsigned long long)__float_as_uint(b) << 32 | __float_as_uint(a), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void take_pair(const unsigned long long *p, float &a, float &b) {
    const unsigned long long v = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    a = __uint_as_float((uint32_t)v);
    b = __uint_as_float((uint32_t)(v >> 32));
}

// Row r of a workgroup's tile: query token r / group of the sequence, q head r % group of the kv head.
struct RowAt {
    size_t q, out;
    bool on;
};
__device__ __forceinline__ RowAt row_at(const CachedArgs &a, int s, int r, int kvh, int group) {
    RowAt x;
    x.on = r < a.q_len * group;
    const int j = x.on ? r / group : 0, h = kvh * group + (x.on ? r % group : 0);
    const size_t token = (size_t)s * a.q_len + j;
    x.q = token * a.q.token_stride + h * a.q.head_stride;
    x.out = token * a.out.token_stride + h * a.out.head_stride;
    return x;
}

// the worker that has unit u (< all) of `active` workers, the last w with w all / active <= u: 32-bit arithmetic where it holds
__device__ __forceinline__ long worker_of(long u, long active, long all) {
    const long n = (u + 1) * active - 1;
    return n <= 0xffffffffl && all <= 0xffffffffl ? (long)((uint32_t)n / (uint32_t)all) : n / all;
}

// Elements 8 l8 .. 8 l8 + 7 of row r of a kv head (the four lanes of a rotation group together): the sums over
// the softmax's total, rotated back.  store: whether there is such a row.
__device__ __forceinline__ void finish_row(const CachedArgs &a, int s, int len, int r, int kvh, int group, int l8, int lane,
                                           bool faulted, bool store, float (&v)[8], float total) {
    const bool sees = len > a.q_len - 1 - r / group;
    const float inv = faulted ? __builtin_nanf("") : (float)(1 << (a.l.bits - 1)) / total;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = sees ? v[e] * inv : 0.f;
    h32_run8(v, lane);
    if (store) store_run8<1>(a.out.data, row_at(a, s, r, kvh, group).out + 8 * l8, a.out.vec, v);
}

// apart: the parts of a sequence that workers share are left for attention_cached_join_kernel.
template <int D, int BITS>
__global__ __launch_bounds__(64 * cached_waves(D)) void attention_cached_kernel(CachedArgs a, void *ws,
                                                                             uint32_t *counts, const uint32_t *status,
                                                                             int workers, size_t slots, int row_tiles, int direct,
                                                                             int apart) {
    using C = Cached<D, BITS>;
    constexpr int kCachedWaves = cached_waves(D);
    constexpr int kPitch = D + 4;  // floats of a row of sums in LDS: rows in different banks
    __shared__ __align__(16) float lds[kCachedWaves * kRows * kPitch + 2 * kCachedWaves * kRows];
    __shared__ int arrived;
    const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.y / row_tiles, row0 = (blockIdx.y - kvh * row_tiles) * kRows;
    const int group = a.q.heads / a.l.kv_heads;
    const int rows = min(kRows, a.q_len * group - row0);  // rows of this tile
    constexpr int kItems = kRows * (D / 8), kThreads = 64 * kCachedWaves, kEach = (kItems + kThreads - 1) / kThreads;
    float qx[kEach][8];
    auto load_q = [&](int s) {  // eight elements of a row per item: row tid / (D / 8), ..
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const int i = tid + n * kThreads, r = i / (D / 8), l8 = i % (D / 8);
#pragma unroll
            for (int e = 0; e < 8; ++e) qx[n][e] = 0.f;
            if (i < kItems && r < rows) load_run8<1>(a.q.data, row_at(a, s, row0 + r, kvh, group).q + 8 * l8, a.q.vec, qx[n]);
        }
    };
    constexpr int kUnit = kTile * kCachedWaves;
    const Share<kUnit> sh{a.kv_lens, (long)a.table_stride * a.l.page_tokens, a.sequences};
    // Lane i's 16-token piece: piece i of the next 64 of this wave, whose tiles are tile0, tile0 + waves, ..
    const int32_t *table = nullptr;
    int page = 0, in_page = 0, id = 0;
    auto look_up = [&](int s, int tile0) {  // asks for its page; table places beyond the last are the last
        table = a.page_table + (size_t)s * a.table_stride;
        const int piece = (tile0 + (lane >> 1) * kCachedWaves) * 2 + (lane & 1), per = a.l.page_tokens / 16;
        page = piece / per;
        in_page = (piece - page * per) * 16;
        id = table[min(page, (int)a.table_stride - 1)];
    };
    int s = 0;
    long unit, last, first = 0, all = 0, active = 0;
    const long w = blockIdx.x;
    if (direct) {
        s = blockIdx.x / (unsigned)direct;
        unit = blockIdx.x - (unsigned)(s * direct);
        last = unit + 1;
        load_q(s);
        look_up(s, (int)unit * kCachedWaves + wave);
    }
    const bool faulted = *status != 0;
    auto zero_rows = [&](int s) {  // a sequence without tokens has no units: its rows are zero
        const float zero[8] = {};
        for (int i = tid; i < rows * (D / 8); i += kThreads)
            store_run8<1>(a.out.data, row_at(a, s, row0 + i / (D / 8), kvh, group).out + 8 * (i % (D / 8)), a.out.vec, zero);
    };
    if (direct) {
        const int units = sh.units(s);
        if (unit == 0 && !units) zero_rows(s);
        if (unit >= units) return;
    } else {
        int longest;
        all = total_units(sh, lane, longest);
        const int each = apart ? 1 : units_each(longest, rows * D);
        active = min((long)workers, (all + each - 1) / each);
        for (int z = (int)w; z < a.sequences; z += workers)
            if (!sh.units(z)) zero_rows(z);
        if (w >= active) return;
        unit = mul_div(w, all, active);
        last = mul_div(w + 1, all, active);
        s = find_unit(sh, unit, lane, first);
    }
    const Parts parts = parts_of(ws, D, min(kRows, a.q_len * group), slots, blockIdx.y);
    _Float16 *const qhi = (_Float16 *)lds, *const qlo = qhi + kRows * D;
    float *const q_unit = (float *)(qlo + kRows * D);         // of each row: 1, or 8 where an eighth is kept
    float *const stat = lds + kCachedWaves * kRows * kPitch;  // (maximum, sum) of [wave][row]
    // the largest score is that of the largest product: a negative scale goes into the queries' signs (and 0 *
    // -infinity, the masked places of a zero scale, must stay -infinity)
    const float c = fmaxf(__builtin_fabsf(a.scale) * kLog2e, 1e-30f), sign = a.scale < 0.f ? -1.f : 1.f;
    const Masks<BITS> masks;
    const typename C::Lane at_lane = C::lane_of(m, g);

    while (unit < last && s < a.sequences) {  // one sequence's part at a time
        const int len = sh.len(s), units = sh.units(s);
        if (!units) {
            ++s;
            continue;
        }
        const int u0 = (int)(unit - first), u1 = (int)(last - first < units ? last - first : units);
        // the first tile is on its way while the queries are prepared
        const int tile_end = (int)((long)u1 * kCachedWaves < (len + kTile - 1) / kTile ? u1 * kCachedWaves
                                                                                      : (len + kTile - 1) / kTile);
        const int halves = (len + 15) / 16;  // 16-token pieces that hold tokens

        // where lane i's piece is: byte offset of its head region, place in the page, and whether its table entry
        // is outside the cache
        uint32_t at_lo = 0, at_hi = 0, place = 0;
        typename C::Half cur[2], nxt[2];
        bool bad_cur[2] = {false, false}, bad_nxt[2] = {false, false};
        int tile0 = u0 * kCachedWaves + wave;
        auto places = [&] {
            const bool on = (tile0 + (lane >> 1) * kCachedWaves) * 2 + (lane & 1) < halves;
            const bool in = id >= 0 && (size_t)id < a.page_count;
            const uint64_t off = (on && in ? (uint64_t)id * a.l.page_bytes : 0) + (uint64_t)kvh * a.l.region;
            at_lo = (uint32_t)off;
            at_hi = (uint32_t)(off >> 32);
            place = on ? (in ? in_page : 0x80000000u) : 0;  // none: the first piece of the first page, masked below
        };
        auto fetch = [&](int tile, typename C::Half (&h)[2], bool (&bad)[2]) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = (tile - tile0) / kCachedWaves * 2 + i;
                const uint32_t lo = __builtin_amdgcn_readlane(at_lo, at), hi = __builtin_amdgcn_readlane(at_hi, at);
                const uint32_t pl = __builtin_amdgcn_readlane(place, at);
                bad[i] = pl >> 31;
                C::load(a.pages + (((uint64_t)hi << 32) | lo), pl & 0x7fffffffu, a.l, at_lane, h[i]);
            }
        };
        const int tile_first = tile0;
        if (tile_first < tile_end) {
            if (!direct) look_up(s, tile0);
            places();
            fetch(tile_first, nxt, bad_nxt);
        }
        // queries: rotated, split in two fp16 parts
        if (!direct) load_q(s);
        __syncthreads();
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const int i = tid + n * kThreads;
            if (i >= kItems) break;  // whole waves
            float large = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) large = fmaxf(large, __builtin_fabsf(qx[n][e]));
            const unsigned long long row_lanes = ((1ull << (D / 8)) - 1) << (lane & ~(D / 8 - 1));
            const bool eighth = __ballot(large > kFullQuery) & row_lanes;
            if (i % (D / 8) == 0) q_unit[i / (D / 8)] = eighth ? 8.f : 1.f;
            const float part = eighth ? sign * 0.125f : sign;
            h32_run8(qx[n], lane);
            h8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                qx[n][e] *= part;
                hi[e] = (_Float16)qx[n][e];
                lo[e] = (_Float16)(qx[n][e] - (float)hi[e]);
            }
            *(h8 *)(qhi + 8 * i) = hi;
            *(h8 *)(qlo + 8 * i) = lo;
        }
        __syncthreads();
        h8 bh[C::NJ], bl[C::NJ];
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) {
            bh[j] = C::q_order(*(const h8 *)(qhi + m * D + g * (D / 4) + 8 * j));
            bl[j] = C::q_order(*(const h8 *)(qlo + m * D + g * (D / 4) + 8 * j));
        }
        const float cq = c * q_unit[m] * (1 << (BITS - 1));
        // keys that this lane's row sees
        const int limit = len - (a.q_len - 1 - (row0 + m) / group);

        f4 o[C::NT];
#pragma unroll
        for (int t = 0; t < C::NT; ++t) o[t] = (f4){0.f, 0.f, 0.f, 0.f};
        float top = kStart, sum = 0.f;
        for (int tile = tile_first; tile < tile_end; tile += kCachedWaves) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                cur[i] = nxt[i];
                bad_cur[i] = bad_nxt[i];
            }
            const int ahead = tile + kCachedWaves;
            if (ahead < tile_end) {
                if (ahead - tile0 >= 32 * kCachedWaves) {
                    tile0 = ahead;
                    look_up(s, tile0);
                    places();
                }
                fetch(ahead, nxt, bad_nxt);
            }
            const int n0 = tile * kTile;
            const bool edge = n0 + kTile > len - (a.q_len - 1);  // some row does not see all of the tile
            if (bad_cur[0] || bad_cur[1]) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (bad_cur[i]) cur[i].ks = 0x7e007e00u;
            }
            bool lost = false;  // a value scale that is not finite in a tile with an edge
            if (edge) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t sc[4] = {cur[i].vs.x & 0xffffu, cur[i].vs.x >> 16, cur[i].vs.y & 0xffffu, cur[i].vs.y >> 16};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool in = n0 + 16 * i + 4 * g + e < len, nan = (sc[e] & 0x7c00u) == 0x7c00u;
                        lost |= in && nan;
                        if (!in || nan) sc[e] = 0;
                    }
                    cur[i].vs = (u2){sc[0] | sc[1] << 16, sc[2] | sc[3] << 16};
                }
            }
            f4 st[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                st[i] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < C::NJ; ++j) {
                    const h8 k = C::key(cur[i], j, masks);
                    st[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, bl[j], st[i], 0, 0, 0);
                    st[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, bh[j], st[i], 0, 0, 0);
                }
            }
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = st[e >> 2][e & 3];
            if (edge) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (n0 + 16 * (e >> 2) + 4 * g + (e & 3) >= limit) x[e] = -INFINITY;
            }
            float best = x[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) best = fmaxf(best, x[e]);
            best *= cq;
            if (__ballot(best > top + kSlack)) {
                const float now = fmaxf(top, over_groups_max(best));
                const float keep = __builtin_amdgcn_exp2f(top - now);
                sum *= keep;
                top = now;
#pragma unroll
                for (int t = 0; t < C::NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[t][e] *= keep;
            }
            h8 p;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], cq, -top));
                sum += v;
                p[e] = (_Float16)v;
            }
#pragma unroll
            for (int t = 0; t < C::NT; ++t) {
                h2 v[4];
                C::value(cur[0], t, v[0], v[1], masks);
                C::value(cur[1], t, v[2], v[3], masks);
                const h8 vt = {v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
                o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, p, o[t], 0, 0, 0);
            }
            if (edge && __ballot(lost)) {  // rare: NaN for the rows that see such a token, in its group's elements
                for (int n = n0; n < n0 + kTile && n < len; ++n) {
                    const int page = n / a.l.page_tokens, id = table[page];
                    if (id < 0 || (size_t)id >= a.page_count) continue;
                    const int off = n - page * a.l.page_tokens;
                    const uint16_t *vs = (const uint16_t *)(a.pages + (size_t)id * a.l.page_bytes + (size_t)kvh * a.l.region +
                                                            a.l.vs_off + (size_t)(off >> 2) * (8 * C::G)) + (off & 3);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint16_t sc = vs[4 * ((4 * g + e) * C::G / 16)];
                        if ((sc & 0x7c00u) == 0x7c00u && n < limit) {
#pragma unroll
                            for (int t = 0; t < C::NT; ++t) o[t][e] = __builtin_nanf("");
                        }
                    }
                }
            }
        }

        // the waves' parts together
        sum = over_groups_sum(sum);
        __syncthreads();
        if (g == 0) {
            stat[(wave * kRows + m) * 2] = top;
            stat[(wave * kRows + m) * 2 + 1] = sum;
        }
        __syncthreads();
        float whole = kStart;
#pragma unroll
        for (int i = 0; i < kCachedWaves; ++i) whole = fmaxf(whole, stat[(i * kRows + m) * 2]);
        const float part = __builtin_amdgcn_exp2f(top - whole);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float *row = lds + (wave * kRows + m) * kPitch + (4 * g + e) * C::NT;
#pragma unroll
            for (int t = 0; t < C::NT; ++t) row[t] = o[t][e] * part;
        }
        __syncthreads();
        // The whole sequence, or a part of it: then the worker that stores the last of the parts sums them, in
        // the workers' order whichever it is.  A part's stores have reached device scope (vmcnt) before its
        // arrival is counted; the count is left zero.
        const long w0 = direct ? 0 : worker_of(first, active, all),
                   w1 = direct ? units - 1 : worker_of(first + units - 1, active, all);
        const bool whole_sequence = w0 == w1;
        const size_t part0 = direct ? (size_t)s * direct : (size_t)s;  // partial of worker 0
        const long me = direct ? unit : w;
        auto finish = [&](int r, int l8, float (&v)[8], float total) {
            finish_row(a, s, len, row0 + r, kvh, group, l8, lane, faulted, r < rows, v, total);
        };
#pragma unroll
        for (int n = 0; n < kEach; ++n) {
            const int i = tid + n * kThreads, r = i / (D / 8), l8 = i % (D / 8);
            if (r >= rows) break;
            float v[8] = {}, peak = kStart, total = 0.f;
#pragma unroll
            for (int k = 0; k < kCachedWaves; ++k) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += lds[(k * kRows + r) * kPitch + 8 * l8 + e];
                peak = fmaxf(peak, stat[(k * kRows + r) * 2]);
            }
#pragma unroll
            for (int k = 0; k < kCachedWaves; ++k)
                total += stat[(k * kRows + r) * 2 + 1] * __builtin_amdgcn_exp2f(stat[(k * kRows + r) * 2] - peak);
            if (whole_sequence || faulted) {
                finish(r, l8, v, total);
            } else {
                const size_t at = (part0 + me) * rows + r;
#pragma unroll
                for (int e = 0; e < 8; e += 2) put_pair(parts.sums + at * (D / 2) + 4 * l8 + e / 2, v[e], v[e + 1]);
                if (l8 == 0) put_pair(parts.stats + at, peak, total);
            }
        }
        if (!whole_sequence && !faulted && !apart) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            uint32_t *count = counts + (size_t)blockIdx.y * a.sequences + s;
            if (tid == 0)
                arrived = (int)__hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            if (arrived == (int)(w1 - w0)) {
                if (tid == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                // four elements each; thread groups take every split-th part, eight of them in flight
                const int items = rows * (D / 4), lanes = items < kThreads ? items : kThreads, split = kThreads / lanes;
                const int grp = tid / lanes;
                for (int i0 = 0; i0 < items; i0 += lanes) {
                    const int i = i0 + tid - grp * lanes, r = i / (D / 4);
                    f4 v = {0.f, 0.f, 0.f, 0.f};
                    float peak = kStart, total = 0.f;
                    if (i < items && grp < split) {
                        for (long k = w0 + grp; k <= w1; k += 8 * split) {
                            f4 x[8];
                            float px[8], tx[8];
#pragma unroll
                            for (int n = 0; n < 8; ++n) {
                                x[n] = (f4){0.f, 0.f, 0.f, 0.f};
                                px[n] = kStart;
                                tx[n] = 0.f;
                                if (k + n * split <= w1) {
                                    const size_t at = (part0 + k + n * split) * rows;
                                    float e[4];
                                    take_pair(parts.stats + at + r, px[n], tx[n]);
                                    take_pair(parts.sums + at * (D / 2) + 2 * i, e[0], e[1]);
                                    take_pair(parts.sums + at * (D / 2) + 2 * i + 1, e[2], e[3]);
                                    x[n] = (f4){e[0], e[1], e[2], e[3]};
                                }
                            }
                            float now = peak;
#pragma unroll
                            for (int n = 0; n < 8; ++n) now = fmaxf(now, px[n]);
                            const float f = __builtin_amdgcn_exp2f(peak - now);
                            v *= f;
                            total *= f;
                            peak = now;
#pragma unroll
                            for (int n = 0; n < 8; ++n) {
                                const float f1 = __builtin_amdgcn_exp2f(px[n] - now);
                                v += x[n] * f1;
                                total += tx[n] * f1;
                            }
                        }
                    }
                    if (split > 1) {
                        f4 *const sums = (f4 *)lds;
                        float *const stats = lds + 4 * kThreads;
                        sums[tid] = v;
                        stats[2 * tid] = peak;
                        stats[2 * tid + 1] = total;
                        __syncthreads();
                        if (grp == 0) {
                            for (int k = 1; k < split; ++k) {
                                const int at = k * lanes + tid;
                                const float now = fmaxf(peak, stats[2 * at]);
                                const float f0 = __builtin_amdgcn_exp2f(peak - now), f1 = __builtin_amdgcn_exp2f(stats[2 * at] - now);
                                peak = now;
                                v = v * f0 + sums[at] * f1;
                                total = total * f0 + stats[2 * at + 1] * f1;
                            }
                        }
                        __syncthreads();
                    }
                    if (i < items && grp == 0) {
                        ((f4 *)lds)[i] = v;
                        if (i % (D / 4) == 0) stat[r] = total;
                    }
                }
                __syncthreads();
                for (int i = tid; i < rows * (D / 8); i += kThreads) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = lds[8 * i + e];
                    finish(i / (D / 8), i % (D / 8), v, stat[i / (D / 8)]);
                }
            }
        }
        unit = first + units;
        first = unit;
        ++s;
    }
}

// One row of a sequence that workers share: workgroup (sequence, row tile, row).  The parts' weights first, then their
// sums, four elements a thread, every split-th part by a group of D / 4 threads.
constexpr int kJoinThreads = 512;
template <int D>
__global__ __launch_bounds__(kJoinThreads) void attention_cached_join_kernel(CachedArgs a, void *ws, const uint32_t *status,
                                                                            int workers, size_t slots, int row_tiles) {
    constexpr int kItems = D / 4, kSplit = kJoinThreads / kItems;
    __shared__ float weight[kCachedGroups], sums[kSplit][D + 4], tops[kJoinThreads / 64], totals[kJoinThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, s = blockIdx.x, r = blockIdx.z;
    const int kvh = blockIdx.y / row_tiles, row0 = (blockIdx.y - kvh * row_tiles) * kRows;
    const int group = a.q.heads / a.l.kv_heads, rows = min(kRows, a.q_len * group - row0);
    if (r >= rows || *status) return;  // a faulted workspace: the rows are NaN already
    const Share<kTile * cached_waves(D)> sh{a.kv_lens, (long)a.table_stride * a.l.page_tokens, a.sequences};
    long all = 0, first = 0;
    for (int s0 = 0; s0 < a.sequences; s0 += 64) {
        const int n = sh.units(s0 + lane), end = wave_scan(n, lane, 64);
        if (s >= s0 && s < s0 + 64) first = all + __builtin_amdgcn_readlane(end - n, s - s0);
        all += __builtin_amdgcn_readlane(end, 63);
    }
    const int len = sh.len(s), units = sh.units(s);
    if (!units) return;
    const long active = min((long)workers, all);
    const long w0 = worker_of(first, active, all);
    const int count = (int)(worker_of(first + units - 1, active, all) - w0) + 1;  // at most kCachedGroups
    if (count == 1) return;  // its worker has stored it
    const Parts parts = parts_of(ws, D, min(kRows, a.q_len * group), slots, blockIdx.y);
    const size_t part0 = (size_t)(s + w0);
    const float2 st = tid < count ? ((const float2 *)parts.stats)[(part0 + tid) * rows + r] : float2{kStart, 0.f};
    auto over_wave = [](float v, auto f) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) v = f(v, __shfl_xor(v, d));
        return v;
    };
    const float top = over_wave(st.x, [](float x, float y) { return fmaxf(x, y); });
    if (lane == 0) tops[tid >> 6] = top;
    __syncthreads();
    float peak = kStart;
#pragma unroll
    for (int i = 0; i < kJoinThreads / 64; ++i) peak = fmaxf(peak, tops[i]);
    const float w = __builtin_amdgcn_exp2f(st.x - peak);
    if (tid < count) weight[tid] = w;
    const float part_total = over_wave(st.y * w, [](float x, float y) { return x + y; });
    if (lane == 0) totals[tid >> 6] = part_total;
    __syncthreads();
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < kJoinThreads / 64; ++i) total += totals[i];
    const int item = tid % kItems, grp = tid / kItems;
    const f4 *x = (const f4 *)parts.sums + (part0 * rows + r) * kItems + item;
    f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int k = grp; k < count; k += kSplit) v += x[(size_t)k * rows * kItems] * weight[k];
    *(f4 *)&sums[grp][4 * item] = v;
    __syncthreads();
    if (tid < 64) {  // whole waves: the rotation exchanges between lanes
        const int l8 = lane % (D / 8);
        float y[8] = {};
        for (int k = 0; k < min(kSplit, count); ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] += sums[k][8 * l8 + e];
        finish_row(a, s, len, row0 + r, kvh, group, l8, lane, false, lane < D / 8, y, total);
    }
}

struct CachedPlan {
    int row_tiles, rows, workers;
    size_t slots;
};
CachedPlan cached_plan(size_t q_heads, size_t kv_heads, size_t sequences, size_t q_len) {
    CachedPlan p;
    const size_t all = q_heads / kv_heads * q_len;
    p.row_tiles = (int)((all + kRows - 1) / kRows);
    p.rows = (int)(all < kRows ? all : kRows);
    const size_t tiles = kv_heads * p.row_tiles;
    p.workers = (int)(tiles < kCachedGroups ? (kCachedGroups + tiles - 1) / tiles : 1);
    p.slots = p.workers + sequences;
    return p;
}

// Whether a second kernel joins the parts of long sequences.  In the first one a single workgroup joins a sequence's,
// so it makes few and long ones (units_each); a kernel of its own costs 4 us and takes as many as there are
// workers.  It pays from about `units` * rows * d^2 = 2^22 (one of a wider head has more to join, and fewer tokens in a
// unit): 16,000 tokens, 4 rows of 256: 18.5 against 26.8 us; 30,723, 5 rows of 256 at 8 bits: 21.4 against 45.9; 16,000, 16
// rows of 128: 16.6 against 19.4; 32,768, 4 rows of 64: 14.1 against 13.1; and not where each sequence has a few
// workers only: 16 of up to 32,768 tokens, 4 rows of 128, 2 workers each: 48.7 against 46.9.  `units` are those
// that the page table has room for: 500 tokens in a table for 32,768, 4 rows of 256: 15.2 against 13.5.
constexpr size_t kApart = (size_t)1 << 22, kApartWorkers = 4;
bool join_apart(size_t units, const CachedPlan &p, size_t d, size_t sequences) {
    return units * p.rows * d * d >= kApart && p.workers >= kApartWorkers * sequences;
}

template <int D>
hipError_t launch_d(const CachedArgs &a, void *workspace, hipStream_t stream) {
    const CachedPlan p = cached_plan(a.q.heads, a.l.kv_heads, a.sequences, a.q_len);
    const size_t tiles = (size_t)a.l.kv_heads * p.row_tiles, unit = (size_t)kTile * cached_waves(D);
    const size_t units = (a.table_stride * a.l.page_tokens + unit - 1) / unit;
    const int direct = units <= (size_t)kDirectUnits && units * a.sequences <= (size_t)p.workers ? (int)units : 0;
    const dim3 grid(direct ? direct * a.sequences : p.workers, (unsigned)tiles);
    void *ws = (uint8_t *)workspace + kSharedPrefixBytes;
    uint32_t *counts = (uint32_t *)workspace, *status = (uint32_t *)((uint8_t *)workspace + kStatusOffset);
    const bool apart = !direct && join_apart(units, p, D, a.sequences);
    const auto kernel = a.l.bits == 4 ? attention_cached_kernel<D, 4> : attention_cached_kernel<D, 8>;
    kernel<<<grid, 64 * cached_waves(D), 0, stream>>>(a, ws, counts, status, p.workers, p.slots, p.row_tiles, direct, apart);
    if (apart)
        attention_cached_join_kernel<D><<<dim3(a.sequences, (unsigned)tiles, p.rows), kJoinThreads, 0, stream>>>(
            a, ws, status, p.workers, p.slots, p.row_tiles);
    return hipGetLastError();
}

}  // namespace

bool attention_cached_fits(size_t q_heads, size_t kv_heads, size_t sequences, size_t q_len) {
    const size_t y = kv_heads * cached_plan(q_heads, kv_heads, sequences, q_len).row_tiles;
    return y <= 65535 && y * sequences * sizeof(uint32_t) <= kGemvExchangeBytes;
}

size_t attention_cached_bytes(size_t q_heads, size_t kv_heads, size_t head_dim, size_t sequences, size_t q_len) {
    const CachedPlan p = cached_plan(q_heads, kv_heads, sequences, q_len);
    return kSharedPrefixBytes + kv_heads * p.row_tiles * part_words(head_dim, p.rows, p.slots) * sizeof(unsigned long long);
}

hipError_t launch_attention_cached(const CachedArgs &a, void *workspace, hipStream_t stream) {
    if (a.l.head_dim == 64) return launch_d<64>(a, workspace, stream);
    if (a.l.head_dim == 128) return launch_d<128>(a, workspace, stream);
    return launch_d<256>(a, workspace, stream);
}

}  // namespace exl3k

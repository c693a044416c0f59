// exl3_attention_prompt.hip -- attention of packed sequences over their own keys and values.
//
// A group of four waves has 128 query rows of one head, 32 per wave, and walks its sequence's
// keys in tiles of KT through two LDS buffers with the running maximum and sum of the softmax.
// A workgroup has one such group, or two that take the even and the odd tiles and are joined
// at the end; few rows over many keys are walked in parts by several workgroups, which a second kernel joins.
// 4 D flops per query and key on mfma_f32_32x32x16_f16, which
// bounds a long prompt.  Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T: a lane's column is one
// query row throughout, so the row's statistics and factors are one register and one exchange
// (lanes l and l ^ 32), and S^T leaves each lane with the weights that it needs as the B
// operand of O^T: keys 8 b + 4 (l / 32) + i of each 32.  V's A operand for those keys is a column of
// the tile, read with ds_read_b64_tr_b16: within 16 lanes it hands lane i the i-th of 16 elements of
// four rows.  16-byte chunks of a row are swizzled so that the rows of one read lie in
// different banks.
// One causal prompt of 8,192 tokens, 32 / 8 heads of 128: 532 to 547 us, 1,005 to 1,034 TFLOP/s, at the 1.63 to 1.69 GHz
// that the chip's power leaves (a large fp16 product: 1,150 to 1,390); seven packed prompts of up to 2,111 tokens, some
// after 500 others, 16 / 4 heads of 64: 47 us, 507 TFLOP/s, bound by waves that are not there (1.2 resident a SIMD on
// average where three fit): the longest sequence has 272 of the 650 workgroups, of up to 41 tiles each, and comes
// last; 37 tokens, 8 / 2 heads of 256: 9.6 us.
#include "exl3_head_rows.hpp"

namespace exl3k {

namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;
typedef __attribute__((address_space(3))) h8 lds_h8;

constexpr int kPromptWaves = 4;  // of a group
constexpr int kPromptRows = 32 * kPromptWaves;  // query rows of a workgroup
// Two groups of waves per workgroup, which share its keys, where one would leave CUs idle and the walk is long:
// one prompt of 3,000 tokens, 8 / 2 heads of 256 (192 workgroups): 80 against 107 us, of 128: 40.9 against
// 49.0; but 300 tokens, 64 / 8 heads of 128 (192 workgroups): 12.5 against 11.5, and seven packed prompts, 16 / 4 heads
// of 64 (650 workgroups): 48.2 against 46.9.
constexpr size_t kTwoGroups = 256, kTwoGroupsKeys = 512;  // at most workgroups, at least keys of a sequence on average
constexpr float kStart = -1e30f;                // running maximum before the first key
constexpr float kSlack = 8.f;                   // scores may pass the running maximum by 2^8
constexpr float kLog2e = 1.4426950408889634f;

// The query tile of a workgroup: tile t counts ceil(rows / kPromptRows) tiles of each sequence
// in turn.  starts that are not ascending or not within the rows count as empty.
struct Span {
    int q0, nq, k0, nk, row0;  // row0: the tile's first row in the sequence; nq = 0: no such tile
};
__device__ __forceinline__ int clamp_to(int v, int top) { return v < 0 ? 0 : (v > top ? top : v); }
__device__ __forceinline__ Span find_tile(const PromptArgs &a, int t, int lane) {
    Span x{};
    int before = 0;
    for (int s0 = 0; s0 < a.sequences; s0 += 64) {
        const int s = s0 + lane < a.sequences ? s0 + lane : a.sequences - 1, left = a.sequences - s0;
        const int q0 = clamp_to(a.q_starts[s], a.q_tokens), q1 = clamp_to(a.q_starts[s + 1], a.q_tokens);
        const int k0 = clamp_to(a.kv_starts[s], a.kv_tokens), k1 = clamp_to(a.kv_starts[s + 1], a.kv_tokens);
        const int n = lane < left && q1 > q0 ? (q1 - q0 + kPromptRows - 1) / kPromptRows : 0;
        int end = n;
        for (int d = 1; d < min(left, 64); d <<= 1) {
            const int o = __shfl_up(end, d);
            end += lane >= d ? o : 0;
        }
        const unsigned long long hit = __ballot(t < before + end);
        if (hit) {
            const int l = __builtin_ctzll(hit);  // the lane and so the span are the wave's
            x.q0 = __builtin_amdgcn_readlane(q0, l);
            x.nq = __builtin_amdgcn_readlane(q1, l) - x.q0;
            x.row0 = (t - before - __builtin_amdgcn_readlane(end - n, l)) * kPromptRows;
            x.k0 = __builtin_amdgcn_readlane(k0, l);
            x.nk = max(0, __builtin_amdgcn_readlane(k1, l) - x.k0);
            return x;
        }
        before += __builtin_amdgcn_readlane(end, min(left, 64) - 1);
    }
    return x;
}

typedef __attribute__((address_space(3))) void lds_void;

template <int D>
struct Prompt {
    static constexpr int KT = D == 256 ? 32 : 64;  // keys of a tile
    static constexpr int CH = D / 8;               // 16-byte chunks of a row
    static constexpr int NS = D / 16;              // MFMA steps over the elements
    static constexpr int NT = D / 32;              // O^T tiles
    static constexpr int PER = KT * CH / (64 * kPromptWaves);  // chunks of each matrix per thread
    static constexpr int RS = 64 * kPromptWaves / CH;          // rows between a thread's chunks

    // Place of chunk c of row r in an LDS tile, in chunks: its own inverse, and the same for rows RS apart (one
    // thread's rows).
    static __device__ __forceinline__ int k_at(int r, int c) {
        return r * CH + (D == 64 ? c ^ ((r >> 1) & 7) : c ^ (r & (RS - 1) & 15));
    }
    static __device__ __forceinline__ int v_at(int r, int c) {
        return r * CH + (D == 64 ? c ^ (((r >> 1) & 1) << 2) : c ^ ((r & 3) << 2));
    }

    // 16 bytes a lane into LDS, in lane order from `to`.  After the builtin of this instruction the compiler has
    // every LDS read wait for the load, since it cannot tell the buffers apart (a prompt of 320 tokens,
    // 12 / 3 heads of 256: 21.5 against 20.6 us).  The load writes no register, takes its address and m0 when it is
    // issued, and m0 is given back: the compiler does not know that it was used.  What it writes in LDS is read
    // after a later step's wait and barrier, and no read between belongs to the buffer that it fills.
    static __device__ __forceinline__ void load_chunk(const char *base, uint32_t at, _Float16 *to) {
        uint32_t m0_was;
        asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                     : "=&s"(m0_was)
                     : "s"((uint32_t)(uintptr_t)(lds_void *)to), "v"(at), "s"(base));
    }
    // Brings the tile at key n0 (keys beyond the last are the last) into an LDS tile; complete after a
    // wait for vmcnt and a barrier.  The loads write LDS directly, 16 bytes a lane in lane order, so the
    // lane takes the chunk that belongs at its place.  NEAR: a tile's rows span less than 2^31 bytes
    // and are 16-byte aligned; else the chunks go through registers.
    template <bool V, bool NEAR>
    static __device__ __forceinline__ void stage(const Heads &m, const _Float16 *base, int n0, int nk, int tid,
                                                 _Float16 *lds) {
        const int r0 = tid / CH, p = tid % CH;
        const int c = (V ? v_at(r0, p) : k_at(r0, p)) - r0 * CH;
        const char *tile = (const char *)(base + (size_t)n0 * m.token_stride);
        if constexpr (NEAR) {
            const uint32_t stride = (uint32_t)m.token_stride * 2;
            _Float16 *const wave_lds = lds + __builtin_amdgcn_readfirstlane(tid >> 6) * 512;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                load_chunk(tile, (uint32_t)min(r0 + i * RS, nk - 1 - n0) * stride + 16 * c, wave_lds + i * (512 * kPromptWaves));
        } else {
            for (int i = 0; i < PER; ++i) {
                const _Float16 *q = (const _Float16 *)tile + (size_t)min(r0 + i * RS, nk - 1 - n0) * m.token_stride + 8 * c;
                h8 t;
#pragma unroll
                for (int e = 0; e < 8; ++e) t[e] = q[e];
                *(h8 *)(lds + 8 * (tid + i * 64 * kPromptWaves)) = t;
            }
        }
    }
    // Chunk i of it where all its rows are there: the thread's offset `at` (offset_in) is the same for every
    // tile, the rest is the scalar base.
    template <bool V>
    static __device__ __forceinline__ uint32_t offset_in(const Heads &m, int tid) {
        const int r0 = tid / CH, p = tid % CH;
        return (uint32_t)r0 * (uint32_t)(m.token_stride * 2) + 16 * ((V ? v_at(r0, p) : k_at(r0, p)) - r0 * CH);
    }
    static __device__ __forceinline__ void stage_chunk(const Heads &m, const _Float16 *base, int n0, int wave, int i,
                                                       uint32_t at, _Float16 *lds) {
        const char *rows = (const char *)(base + (size_t)(n0 + i * RS) * m.token_stride);
        load_chunk(rows, at, lds + wave * 512 + i * (512 * kPromptWaves));
    }
};

__device__ __forceinline__ float other_half(float v) {  // the value of lane l ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return __int_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// whether any half of the chunk is infinite or NaN; those become 0
__device__ __forceinline__ bool drop_non_finite(h8 &v) {
    u4 w = bitcast<u4>(v);
    bool found = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & 0x7c00u) == 0x7c00u) {
            w[i] &= 0xffff0000u;
            found = true;
        }
        if ((w[i] & 0x7c000000u) == 0x7c000000u) {
            w[i] &= 0xffffu;
            found = true;
        }
    }
    v = bitcast<h8>(w);
    return found;
}

// Four elements of a row, 32 t + 8 b + 4 h on, where h is the lane's half and j = 4 t + b.
__device__ __forceinline__ void store_out(const PromptArgs &a, const Span &sp, int head, int row, int j, int h, const h4 &x) {
    _Float16 *at = (_Float16 *)a.out.data + (size_t)(sp.q0 + row) * a.out.token_stride + head * a.out.head_stride + 8 * j + 4 * h;
    if (a.out.vec) {
        *(h4 *)at = x;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) at[e] = x[e];
    }
}
// Workgroup b runs on XCD b % 8, each with its own L2: where the heads divide by 8, an XCD takes
// neighbouring heads, which share keys and values (8,192 tokens, 32 / 8 heads of 128: 575 against 580 us).
__device__ __forceinline__ int head_of(const PromptArgs &a, unsigned block) {
    const int place = block % a.q.heads;
    return a.q.heads % 8 ? place : place % 8 * (a.q.heads / 8) + place / 8;
}
// keys that row r of the sequence sees
__device__ __forceinline__ int seen_by(const PromptArgs &a, const Span &sp, int r) {
    const int n = a.causal ? (r < sp.nq ? r : sp.nq - 1) + sp.nk - sp.nq + 1 : sp.nk;
    return n < 0 ? 0 : n;
}
// tiles of a part of a walk of `all` tiles
__device__ __forceinline__ int part_tiles(int all, int parts) { return (all + parts - 1) / parts; }
// floats of a part: f4 [D / 8][thread] sums, then (maximum, sum) [thread]
template <int D>
constexpr size_t kPartFloats = 64 * kPromptWaves * (D / 2 + 2);

// SPLIT: workgroup (b, i) walks part i of the keys and leaves its sums in `ws` for attention_prompt_join_kernel.
template <int D, bool NEAR, int kGroups, bool SPLIT>
__global__ __launch_bounds__(64 * kPromptWaves * kGroups, 2) void attention_prompt_kernel(PromptArgs a, int tiles, float *ws) {
    using P = Prompt<D>;
    constexpr int KT = P::KT;
    __shared__ __align__(1024) _Float16 tile_lds[2][kGroups][2][KT * D];  // keys, values; of each group two buffers
    const int tid = threadIdx.x % (64 * kPromptWaves), lane = tid & 63, m = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = __builtin_amdgcn_readfirstlane(threadIdx.x / (64 * kPromptWaves));
    auto &ks = tile_lds[0][group], &vs = tile_lds[1][group];
    const int head = head_of(a, blockIdx.x);
    const Span sp = find_tile(a, tiles - 1 - (int)(blockIdx.x / a.q.heads), lane);  // a causal sequence's longest first
    if (!sp.nq) return;
    const int kvh = head / (a.q.heads / a.k.heads);
    const _Float16 *kb = (const _Float16 *)a.k.data + (size_t)sp.k0 * a.k.token_stride + kvh * a.k.head_stride;
    const _Float16 *vb = (const _Float16 *)a.v.data + (size_t)sp.k0 * a.v.token_stride + kvh * a.v.head_stride;

    // keys that this lane's row, the wave's last row and the workgroup's last row see
    const int row = sp.row0 + 32 * wave + m;
    const int limit = seen_by(a, sp, row);
    const int last = seen_by(a, sp, sp.row0 + kPromptRows - 1);
    const int all = (last + KT - 1) / KT;  // tiles of the walk; this workgroup's are lo .. lo + steps - 1
    int lo = 0, steps = all;
    if constexpr (SPLIT) {
        const int per = part_tiles(all, gridDim.y);
        lo = min((int)blockIdx.y * per, all);
        steps = min(per, all - lo);
        if (!steps) return;
    }
    const int end = (lo + steps) * KT;
    const int wave_end = min(seen_by(a, sp, sp.row0 + 32 * wave + 31), end);
    const int q_row = row < sp.nq ? row : sp.nq - 1;
    const _Float16 *qp = (const _Float16 *)a.q.data + (size_t)(sp.q0 + q_row) * a.q.token_stride + head * a.q.head_stride;
    h8 q[P::NS];
#pragma unroll
    for (int s = 0; s < P::NS; ++s) {
        if (a.q.vec) {
            q[s] = *(const h8 *)(qp + 16 * s + 8 * h);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) q[s][e] = qp[16 * s + 8 * h + e];
        }
    }
    f16v o[P::NT];
#pragma unroll
    for (int t = 0; t < P::NT; ++t)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[t][e] = 0.f;
    float top = kStart, sum = 0.f;  // top: the running maximum, as a score times c
    // the largest score is that of the largest product: a negative scale goes into the queries' signs (and
    // 0 * -infinity, the masked places of a zero scale, must stay -infinity)
    if (a.scale < 0.f) {
#pragma unroll
        for (int s = 0; s < P::NS; ++s) q[s] = -q[s];
    }
    const float c = fmaxf(__builtin_fabsf(a.scale) * kLog2e, 1e-30f);

    // Where the lane reads in a tile, in bytes: a chunk index enters its swizzle as an exclusive or of whole
    // bits, so chunk 2 s + h of a key is k_lane ^ 32 s and tile t of a value v_lane ^ 64 t; rows 16 on are
    // constant offsets.
    const int k_lane = 16 * P::k_at(m, h);
    const int li = lane & 15;
    const int v_lane = 16 * P::v_at(4 * h + (li >> 2), 2 * ((lane >> 4) & 1) + ((li & 3) >> 1)) + 8 * (li & 1);
    // tiles of this workgroup without a masked place
    const int whole = max(0, min(seen_by(a, sp, sp.row0) / KT - lo, steps));

    f16v st[KT / 32];  // a tile's scores
    h8 p[KT / 16];
    // operands from LDS: MFMA n of a tile's scores, MFMA n of its weighted values
    auto key_frag = [&](int kt, int n) {
        return *(const lds_h8 *)(uint32_t)((kt ^ (n % P::NS * 32)) + n / P::NS * 64 * D);
    };
    auto value_frag = [&](int vt, int n) {
        const uint32_t at = (uint32_t)((vt ^ (n % P::NT * 64)) + n / P::NT * 32 * D);
        const h4 lo = bitcast<h4>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)at));
        const h4 hi = bitcast<h4>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(at + 16 * D)));
        return (h8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    const int k_base = (int)(uintptr_t)(lds_void *)ks[0] + k_lane, v_base = (int)(uintptr_t)(lds_void *)vs[0] + v_lane;
    constexpr int kBuf = KT * D * 2;  // bytes of a buffer
    auto score = [&](int n, h8 k) {
        const f16v zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        st[n / P::NS] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[n % P::NS], n % P::NS ? st[n / P::NS] : zero, 0, 0, 0);
    };
    auto add_value = [&](int n, h8 v) {
        o[n % P::NT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[n / P::NT], o[n % P::NT], 0, 0, 0);
    };
    // two weights, rounded to fp16 for the product; the sum is that of the rounded ones
    auto weigh = [&](int j) {
        const int b = j / 8, e = j % 8 * 2;
        const h2 w = {(_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(st[b][e], c, -top)),
                      (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(st[b][e + 1], c, -top))};
        sum = __builtin_amdgcn_fdot2(w, (h2){(_Float16)1.f, (_Float16)1.f}, sum, false);
        p[2 * b + e / 8][e % 8] = w[0];
        p[2 * b + e / 8][e % 8 + 1] = w[1];
    };
    // the running maximum moves only when a score passes it by kSlack
    auto raise = [&](float best) {
        best *= c;
        if (__ballot(best > top + kSlack)) {
            const float now = fmaxf(top, fmaxf(best, other_half(best)));
            const float keep = __builtin_amdgcn_exp2f(top - now);
            sum *= keep;
            top = now;
#pragma unroll
            for (int t = 0; t < P::NT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[t][e] *= keep;
        }
    };
    auto largest = [&] {
        float best = st[0][0];
#pragma unroll
        for (int b = 0; b < KT / 32; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) best = fmaxf(best, st[b][e]);
        return best;
    };
    constexpr int kMfma = KT / 32 * P::NS, kPairs = KT / 4;  // MFMAs of each product, pairs of weights
    static_assert(kMfma == KT / 16 * P::NT, "both products take as many MFMAs");
    // Step i of a group is tile lo + 2 i + group.  It ends with the scores of step i + 1.  Its tiles (keys of
    // step i + 1, values of step i) were asked for in step i - 1; it asks for the keys of i + 2 and the values of
    // i + 1 in the buffers that step i - 1 was done with.
    auto key_of = [&](int i) { return (lo + i * kGroups + group) * KT; };  // a step's first key
    auto next = [&](int i) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (key_of(i + 2) < end) P::template stage<false, NEAR>(a.k, kb, key_of(i + 2), sp.nk, tid, ks[i & 1]);
        if (key_of(i + 1) < end) P::template stage<true, NEAR>(a.v, vb, key_of(i + 1), sp.nk, tid, vs[(i + 1) & 1]);
    };
    const int rounds = (steps + kGroups - 1) / kGroups;
    if (key_of(0) < end) {
        P::template stage<false, NEAR>(a.k, kb, key_of(0), sp.nk, tid, ks[0]);
        P::template stage<true, NEAR>(a.v, vb, key_of(0), sp.nk, tid, vs[0]);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (key_of(1) < end) P::template stage<false, NEAR>(a.k, kb, key_of(1), sp.nk, tid, ks[1]);
#pragma unroll
    for (int n = 0; n < kMfma; ++n) score(n, key_frag(k_base, n));  // without a tile: not used
    // Tiles without masked places, while the tiles to ask for have all their rows.
    const uint32_t k_at = P::template offset_in<false>(a.k, tid), v_at = P::template offset_in<true>(a.v, tid);
    // At least one step is left to the loop after: its wait ends the loads under way.
    const int plain = NEAR ? min(min(whole / kGroups, rounds - 1), (sp.nk / KT - lo) / kGroups - 2) : 0;
    auto ask_chunk = [&](int i, int n) {  // of the keys of step i + 2 and the values of step i + 1, in turn
        if (n % 2 == 0) P::stage_chunk(a.k, kb, key_of(i + 2), wave, n / 2, k_at, ks[i & 1]);
        else P::stage_chunk(a.v, vb, key_of(i + 1), wave, n / 2, v_at, vs[(i + 1) & 1]);
    };
    // A tile's weights free its scores' registers for the next tile's, whose MFMAs and those of the values follow
    // with the loads between them (asked for at once they hold the wave for 650 cycles: 32 KB at the 64 bytes a
    // clock of a CU's address path); the exponentials run beside the other waves' MFMAs.  Two tiles of scores
    // in flight, or an order fixed by hand, gained nothing more: 597 against 600 us then at 8,192 tokens of 32 / 8
    // heads of 128, which runs into the power limit (the MFMAs alone: 400 us).
    int i = 0;
    float best = largest();
    for (; i < plain; ++i) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        raise(best);
        int kt = k_base + ((i + 1) & 1) * kBuf, vt = v_base + (i & 1) * kBuf;
        asm volatile("" : "+v"(kt), "+v"(vt));  // else every read's address is kept across the loop, and operands spilt
#pragma unroll
        for (int j = 0; j < kPairs; ++j) weigh(j);
#pragma unroll
        for (int n = 0; n < kMfma; ++n) {
            score(n, key_frag(kt, n));
            if (n % (kMfma / P::PER) == 0) ask_chunk(i, 2 * n / (kMfma / P::PER));
        }
#pragma unroll
        for (int n = 0; n < kMfma; ++n) {
            add_value(n, value_frag(vt, n));
            if (n % (kMfma / P::PER) == 0) ask_chunk(i, 2 * n / (kMfma / P::PER) + 1);
        }
        best = largest();
    }
    __shared__ int odd_tile[2];  // whether the step's values held a non-finite one
    if (threadIdx.x < 2) odd_tile[threadIdx.x] = 0;
    for (; i < rounds; ++i) {  // the others
        const int n0 = key_of(i);
        next(i);
        // a masked value must not reach a row: 0 * NaN.  Non-finite values are taken out of the tile here
        // and added below for the rows that see them.
        bool odd = false;
        if (i >= whole / kGroups) {
            for (int j = 0; j < P::PER && n0 < end; ++j) {
                h8 *const at = (h8 *)(vs[i & 1]) + tid + j * 64 * kPromptWaves;
                h8 v = *at;
                if (drop_non_finite(v)) {
                    *at = v;
                    odd = true;
                }
            }
            if (__ballot(odd) && lane == 0) odd_tile[i & 1] = 1;
            __syncthreads();
            odd = odd_tile[i & 1];
            if (threadIdx.x == 0) odd_tile[(i + 1) & 1] = 0;
        }
        if (n0 < wave_end) {  // else no row of this wave sees the tile, or there is none
#pragma unroll
            for (int b = 0; b < KT / 32; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    st[b][e] = n0 + 32 * b + 8 * (e >> 2) + 4 * h + (e & 3) < limit ? st[b][e] : -INFINITY;
            raise(largest());
#pragma unroll
            for (int j = 0; j < kPairs; ++j) weigh(j);
#pragma unroll
            for (int n = 0; n < kMfma; ++n) add_value(n, value_frag(v_base + (i & 1) * kBuf, n));
            if (odd) {  // rare
                for (int n = n0; n < n0 + KT && n < sp.nk; ++n) {
                    const _Float16 *vr = vb + (size_t)n * a.v.token_stride;
#pragma unroll
                    for (int t = 0; t < P::NT; ++t)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float x = (float)vr[32 * t + 8 * (e >> 2) + 4 * h + (e & 3)];
                            if (!__builtin_isfinite(x) && n < limit) o[t][e] += x;
                        }
                }
            }
            if (key_of(i + 1) < end) {
#pragma unroll
                for (int n = 0; n < kMfma; ++n) score(n, key_frag(k_base + ((i + 1) & 1) * kBuf, n));
            }
        }
    }
    if constexpr (kGroups == 2) {
        // the odd tiles' part into the even ones', register by register of the same lane
        __shared__ float stats[2][64 * kPromptWaves];
        f4 *const parts = (f4 *)tile_lds;  // 16 NT floats a lane: half of the tiles' LDS, at head dimension 256 all of it
        static_assert(sizeof(tile_lds) >= 64 * kPromptWaves * 16 * P::NT * sizeof(float), "the tiles' LDS holds a group's sums");
        __syncthreads();
        if (group == 1) {
            stats[0][tid] = top;
            stats[1][tid] = sum;
    #pragma unroll
            for (int t = 0; t < P::NT; ++t)
    #pragma unroll
                for (int b = 0; b < 4; ++b)
                    parts[(4 * t + b) * (64 * kPromptWaves) + tid] = (f4){o[t][4 * b], o[t][4 * b + 1], o[t][4 * b + 2], o[t][4 * b + 3]};
        }
        __syncthreads();
        if (group == 1) return;
        const float other = stats[0][tid], peak = fmaxf(top, other);
        const float mine = __builtin_amdgcn_exp2f(top - peak), theirs = __builtin_amdgcn_exp2f(other - peak);
        sum = sum * mine + stats[1][tid] * theirs;
        top = peak;
    #pragma unroll
        for (int t = 0; t < P::NT; ++t)
    #pragma unroll
            for (int b = 0; b < 4; ++b) {
                const f4 x = parts[(4 * t + b) * (64 * kPromptWaves) + tid];
    #pragma unroll
                for (int e = 0; e < 4; ++e) o[t][4 * b + e] = o[t][4 * b + e] * mine + x[e] * theirs;
            }
    }
    sum += other_half(sum);
    if (row >= sp.nq) return;
    if constexpr (SPLIT) {
        f4 *const part = (f4 *)(ws + ((size_t)blockIdx.x * gridDim.y + blockIdx.y) * kPartFloats<D>);
#pragma unroll
        for (int j = 0; j < 4 * P::NT; ++j)
            part[j * (64 * kPromptWaves) + tid] = (f4){o[j / 4][j % 4 * 4], o[j / 4][j % 4 * 4 + 1], o[j / 4][j % 4 * 4 + 2], o[j / 4][j % 4 * 4 + 3]};
        ((float2 *)(part + 4 * P::NT * (64 * kPromptWaves)))[tid] = float2{top, sum};
        return;
    }
    const float inv = limit > 0 ? 1.0f / sum : 0.f;
#pragma unroll
    for (int j = 0; j < 4 * P::NT; ++j) {
        h4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (_Float16)(limit > 0 ? o[j / 4][j % 4 * 4 + e] * inv : 0.f);
        store_out(a, sp, head, row, j, h, x);
    }
}

// The parts of each row together, in their order: thread tid of workgroup (b, i) has the elements that lane tid of
// workgroups (b, part) had in their sums 4 i .. 4 i + 3.
template <int D>
__global__ __launch_bounds__(64 * kPromptWaves) void attention_prompt_join_kernel(PromptArgs a, int tiles, const float *ws,
                                                                               int parts) {
    constexpr int kThreads = 64 * kPromptWaves;
    const int tid = threadIdx.x, lane = tid & 63;
    const Span sp = find_tile(a, tiles - 1 - (int)(blockIdx.x / a.q.heads), lane);
    const int row = sp.row0 + 32 * (tid >> 6) + (lane & 31);
    if (row >= sp.nq) return;
    const int all = (seen_by(a, sp, sp.row0 + kPromptRows - 1) + Prompt<D>::KT - 1) / Prompt<D>::KT;
    const int some = all ? (all + part_tiles(all, parts) - 1) / part_tiles(all, parts) : 0;  // parts with tiles
    const bool sees = seen_by(a, sp, row) > 0;
    const f4 *part = (const f4 *)(ws + (size_t)blockIdx.x * parts * kPartFloats<D>);
    constexpr size_t kStep = kPartFloats<D> / 4;
    auto stats = [&](int i) { return ((const float2 *)(part + i * kStep + D / 8 * kThreads))[tid]; };
    float peak = kStart, total = 0.f;
#pragma unroll 8
    for (int i = 0; i < some; ++i) peak = fmaxf(peak, stats(i).x);
    f4 v[4] = {};
    const f4 *mine = part + blockIdx.y * 4 * kThreads + tid;
#pragma unroll 4
    for (int i = 0; i < some; ++i) {
        const float2 st = stats(i);
        const float w = __builtin_amdgcn_exp2f(st.x - peak);
        total += st.y * w;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += mine[i * kStep + j * kThreads] * w;
    }
    const float inv = 1.0f / total;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        h4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (_Float16)(sees ? v[j][e] * inv : 0.f);
        store_out(a, sp, head_of(a, blockIdx.x), row, blockIdx.y * 4 + j, lane >> 5, x);
    }
}

int prompt_tiles(int q_tokens, int sequences) { return q_tokens / kPromptRows + sequences; }  // each may end in a part tile

// Parts of a walk.  Where the workgroups leave CUs idle, parts of the keys go to them, one workgroup a CU, and a
// second kernel joins the parts.  A round of two tiles takes 1.3 us, the join 4 us and 0.3 us a part more, so
// r rounds are best cut in about 2 sqrt(r), and the cut has to save 5 of them: 16 tokens after 8,192 others,
// 32 / 8 heads of 128: 26.9 against 94.9 us (8 parts), 8 / 2 heads of 256: 30.2 against 194.7 (16); 1,000 tokens,
// 4 / 1 heads of 128: 16.0 against 20.4 (5); 2,000 tokens, 8 / 2 heads of 256: 49.0 against 58.9 (2); but four prompts of 300 after 256 others: 16.1 against 15.1 (4).
// More workgroups than CUs: 2,000 tokens, 4 / 1 heads of 128: 28.6 us at 6 parts, 20.4 at 4.
constexpr size_t kSplitGroups = 256, kSplitGain = 5;
int prompt_parts(size_t q_heads, int head_dim, int sequences, int q_tokens, int kv_tokens) {
    const size_t groups = (size_t)prompt_tiles(q_tokens, sequences) * q_heads, idle = kSplitGroups / groups;
    const size_t round = 2 * (head_dim == 256 ? Prompt<256>::KT : head_dim == 128 ? Prompt<128>::KT : Prompt<64>::KT);
    const size_t rounds = (size_t)kv_tokens / sequences / round;
    size_t parts = 1;
    while (parts < idle && parts * parts < 4 * rounds) ++parts;
    return rounds * (parts - 1) >= kSplitGain * parts ? (int)parts : 1;
}

template <int D, bool NEAR>
void launch_near(const PromptArgs &a, float *workspace, hipStream_t stream) {
    const int tiles = prompt_tiles(a.q_tokens, a.sequences), block = 64 * kPromptWaves;
    const unsigned groups = (unsigned)tiles * a.q.heads;
    const int parts = prompt_parts(a.q.heads, D, a.sequences, a.q_tokens, a.kv_tokens);
    if (parts > 1) {
        attention_prompt_kernel<D, NEAR, 2, true><<<dim3(groups, parts), 2 * block, 0, stream>>>(a, tiles, workspace);
        attention_prompt_join_kernel<D><<<dim3(groups, D / 32), block, 0, stream>>>(a, tiles, workspace, parts);
    } else if (groups <= kTwoGroups && (size_t)a.kv_tokens >= kTwoGroupsKeys * a.sequences) {
        attention_prompt_kernel<D, NEAR, 2, false><<<groups, 2 * block, 0, stream>>>(a, tiles, nullptr);
    } else {
        attention_prompt_kernel<D, NEAR, 1, false><<<groups, block, 0, stream>>>(a, tiles, nullptr);
    }
}

template <int D>
hipError_t launch_d(const PromptArgs &a, void *workspace, hipStream_t stream) {
    constexpr size_t kNear = (size_t)1 << 31;
    const bool near = a.k.vec && a.v.vec && a.k.token_stride * (2 * Prompt<D>::KT) < kNear &&
                      a.v.token_stride * (2 * Prompt<D>::KT) < kNear;
    float *const ws = workspace ? (float *)((uint8_t *)workspace + kSharedPrefixBytes) : nullptr;
    if (near) launch_near<D, true>(a, ws, stream);
    else launch_near<D, false>(a, ws, stream);
    return hipGetLastError();
}

}  // namespace

size_t attention_prompt_bytes(size_t q_heads, int head_dim, int sequences, int q_tokens, int kv_tokens) {
    const size_t parts = prompt_parts(q_heads, head_dim, sequences, q_tokens, kv_tokens);
    if (parts < 2) return 0;
    return kSharedPrefixBytes + prompt_tiles(q_tokens, sequences) * q_heads * parts * 64 * kPromptWaves * (head_dim / 2 + 2) * sizeof(float);
}

hipError_t launch_attention_prompt(const PromptArgs &a, void *workspace, hipStream_t stream) {
    if (a.head_dim == 64) return launch_d<64>(a, workspace, stream);
    if (a.head_dim == 128) return launch_d<128>(a, workspace, stream);
    return launch_d<256>(a, workspace, stream);
}

}  // namespace exl3k

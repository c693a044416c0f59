// exl3_attention_prompt.hip -- attention of packed sequences over their own keys and values.
//
// A workgroup of four waves has 128 query rows of one head, 32 per wave, and walks its
// sequence's keys in tiles of KT through two LDS buffers, with the running maximum and sum of
// the softmax: 4 D flops per query and key on mfma_f32_32x32x16_f16, which bounds a long
// prompt.  Both products are taken transposed, S^T = K Q^T and O^T = V^T P^T: a lane's column is one
// query row throughout, so the row's statistics and factors are one register and one exchange
// (lanes l and l ^ 32), and S^T leaves each lane with the weights that it needs as the B
// operand of O^T: keys 8 b + 4 (l / 32) + i of each 32.  V's A operand for those keys is a column of
// the tile, read with ds_read_b64_tr_b16: within 16 lanes it hands lane i the i-th of 16 elements of
// four rows.  16-byte chunks of a row are swizzled so that the rows of one read lie in
// different banks.
#include "exl3_head_rows.hpp"

namespace exl3k {

namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

constexpr int kPromptWaves = 4;
constexpr int kPromptRows = 32 * kPromptWaves;  // query rows of a workgroup
constexpr float kStart = -1e30f;                // running maximum before the first key
constexpr float kSlack = 8.f;                   // scores may pass the running maximum by 2^8
constexpr float kLog2e = 1.4426950408889634f;

// The query tile of a workgroup: tile t counts ceil(rows / kPromptRows) tiles of each sequence
// in turn.  starts that are not ascending or not within the rows count as empty.
struct Span {
    int q0, nq, k0, nk, row0;  // row0: the tile's first row in the sequence; nq = 0: no such tile
};
__device__ __forceinline__ int clamp_to(int v, int top) { return v < 0 ? 0 : (v > top ? top : v); }
__device__ __forceinline__ int rows_of(const PromptArgs &a, int s) {
    if (s >= a.sequences) return 0;
    const int b = clamp_to(a.q_starts[s], a.q_tokens), e = clamp_to(a.q_starts[s + 1], a.q_tokens);
    return e > b ? e - b : 0;
}
__device__ __forceinline__ Span find_tile(const PromptArgs &a, int t, int lane) {
    Span x{};
    int before = 0;
    for (int s0 = 0; s0 < a.sequences; s0 += 64) {
        const int n = (rows_of(a, s0 + lane) + kPromptRows - 1) / kPromptRows;
        int end = n;
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(end, d);
            end += lane >= d ? o : 0;
        }
        const unsigned long long hit = __ballot(t < before + end);
        if (hit) {
            const int l = __builtin_ctzll(hit), s = s0 + l;
            x.q0 = clamp_to(a.q_starts[s], a.q_tokens);
            x.nq = rows_of(a, s);
            x.row0 = (t - before - __shfl(end - n, l)) * kPromptRows;
            x.k0 = clamp_to(a.kv_starts[s], a.kv_tokens);
            x.nk = clamp_to(a.kv_starts[s + 1], a.kv_tokens) - x.k0;
            if (x.nk < 0) x.nk = 0;
            return x;
        }
        before += __shfl(end, 63);
    }
    return x;
}

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

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

    // Brings the tile at key n0 (keys beyond the last are the last) into an LDS tile; complete after a
    // wait for vmcnt and a barrier.  The loads write LDS directly, 16 bytes a lane in lane order, so the
    // lane takes the chunk that belongs at its place.  `near`: a tile's rows span less than 2^31 bytes
    // and are 16-byte aligned; else the chunks go through registers.
    template <bool V>
    static __device__ __forceinline__ void stage(const Heads &m, const _Float16 *base, bool near, int n0, int nk, int tid,
                                                 _Float16 *lds) {
        const int r0 = tid / CH, p = tid % CH;
        const int c = (V ? v_at(r0, p) : k_at(r0, p)) - r0 * CH;
        const char *tile = (const char *)(base + (size_t)n0 * m.token_stride);
        if (near) {
            const uint32_t stride = (uint32_t)m.token_stride * 2;
            _Float16 *const wave_lds = lds + __builtin_amdgcn_readfirstlane(tid >> 6) * 512;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                __builtin_amdgcn_global_load_lds(
                    (global_void *)(tile + ((uint32_t)min(r0 + i * RS, nk - 1 - n0) * stride + 16 * c)),
                    (lds_void *)(wave_lds + i * (512 * kPromptWaves)), 16, 0, 0);
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

template <int D>
__global__ __launch_bounds__(64 * kPromptWaves, 2) void attention_prompt_kernel(PromptArgs a, int tiles) {
    using P = Prompt<D>;
    constexpr int KT = P::KT;
    __shared__ __align__(16) _Float16 ks[2][KT * D], vs[2][KT * D];
    const int tid = threadIdx.x, lane = tid & 63, m = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int head = blockIdx.x % a.q.heads;
    const Span sp = find_tile(a, tiles - 1 - (int)(blockIdx.x / a.q.heads), lane);  // a causal sequence's longest first
    if (!sp.nq) return;
    const int kvh = head / (a.q.heads / a.k.heads);
    const _Float16 *kb = (const _Float16 *)a.k.data + (size_t)sp.k0 * a.k.token_stride + kvh * a.k.head_stride;
    const _Float16 *vb = (const _Float16 *)a.v.data + (size_t)sp.k0 * a.v.token_stride + kvh * a.v.head_stride;

    // keys that this lane's row, the wave's last row and the workgroup's last row see
    const int row = sp.row0 + 32 * wave + m;
    const int shift = a.causal ? sp.nk - sp.nq + 1 : 0;
    auto seen = [&](int r) {
        const int n = a.causal ? (r < sp.nq ? r : sp.nq - 1) + shift : sp.nk;
        return n < 0 ? 0 : n;
    };
    const int limit = seen(row);
    const int wave_max_ = seen(sp.row0 + 32 * wave + 31);
    const int last = seen(sp.row0 + kPromptRows - 1);
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

    const bool k_near = a.k.vec && a.k.token_stride * (2 * KT) < ((size_t)1 << 31);
    const bool v_near = a.v.vec && a.v.token_stride * (2 * KT) < ((size_t)1 << 31);
    // Where the lane reads in a tile: the swizzles repeat every 16 rows, so rows further on are constant
    // offsets.
    int k_lane[P::NS], v_lane[P::NT];
#pragma unroll
    for (int s = 0; s < P::NS; ++s) k_lane[s] = 8 * P::k_at(m, 2 * s + h);
#pragma unroll
    for (int t = 0; t < P::NT; ++t) {
        const int i = lane & 15;
        v_lane[t] = 8 * P::v_at(4 * h + (i >> 2), 4 * t + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) + 4 * (i & 1);
    }
    const int steps = (last + KT - 1) / KT;
    const int open = seen(sp.row0);
    const int whole = open / KT < steps ? open / KT : steps;  // tiles without a masked place

    f16v st[KT / 32], ahead[KT / 32];
    h8 p[KT / 16];
    auto scores = [&](const _Float16 *kt, f16v (&x)[KT / 32]) {
#pragma unroll
        for (int b = 0; b < KT / 32; ++b) {
#pragma unroll
            for (int e = 0; e < 16; ++e) x[b][e] = 0.f;
#pragma unroll
            for (int s = 0; s < P::NS; ++s)
                x[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const h8 *)(kt + k_lane[s] + b * 32 * D), q[s], x[b], 0, 0, 0);
        }
    };
    // the running maximum moves only when a score passes it by kSlack
    auto raise = [&] {
        float best = st[0][0];
#pragma unroll
        for (int b = 0; b < KT / 32; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) best = fmaxf(best, st[b][e]);
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
    // weights, rounded to fp16 for the product; the sum is that of the rounded ones
    auto weigh = [&] {
#pragma unroll
        for (int b = 0; b < KT / 32; ++b)
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const h2 w = {(_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(st[b][e], c, -top)),
                              (_Float16)__builtin_amdgcn_exp2f(__builtin_fmaf(st[b][e + 1], c, -top))};
                sum = __builtin_amdgcn_fdot2(w, (h2){(_Float16)1.f, (_Float16)1.f}, sum, false);
                p[2 * b + e / 8][e % 8] = w[0];
                p[2 * b + e / 8][e % 8 + 1] = w[1];
            }
    };
    auto add_values = [&](const _Float16 *vt) {
#pragma unroll
        for (int u = 0; u < KT / 16; ++u)
#pragma unroll
            for (int t = 0; t < P::NT; ++t) {
                const _Float16 *at = vt + v_lane[t] + u * 16 * D;
                const h4 lo = bitcast<h4>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)at));
                const h4 hi = bitcast<h4>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(at + 8 * D)));
                const h8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[u], o[t], 0, 0, 0);
            }
    };
    // Step i ends with the scores of tile i + 1, so their MFMAs and the exponentials of tile i share it.
    // Its tiles (keys i + 1, values i) were asked for in step i - 1; it asks for keys i + 2 and values
    // i + 1 in the buffers that step i - 1 was done with.
    auto next = [&](int i) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (i + 2 < steps) P::template stage<false>(a.k, kb, k_near, (i + 2) * KT, sp.nk, tid, ks[i & 1]);
        if (i + 1 < steps) P::template stage<true>(a.v, vb, v_near, (i + 1) * KT, sp.nk, tid, vs[(i + 1) & 1]);
    };
    if (steps) {
        P::template stage<false>(a.k, kb, k_near, 0, sp.nk, tid, ks[0]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (steps > 1) P::template stage<false>(a.k, kb, k_near, KT, sp.nk, tid, ks[1]);
        P::template stage<true>(a.v, vb, v_near, 0, sp.nk, tid, vs[0]);
        scores(ks[0], st);
    }
    for (int i = 0; i < whole; ++i) {
        next(i);
        raise();
        scores(ks[(i + 1) & 1], ahead);  // after the last tile: of no use, and not used
        weigh();
        add_values(vs[i & 1]);
#pragma unroll
        for (int b = 0; b < KT / 32; ++b) st[b] = ahead[b];
    }
    for (int i = whole; i < steps; ++i) {  // tiles with masked places
        const int n0 = i * KT;
        next(i);
        // a masked value must not reach a row: 0 * NaN.  Non-finite values are taken out of the tile here
        // and added below for the rows that see them.
        bool odd = false;
        for (int j = 0; j < P::PER; ++j) {
            h8 *const at = (h8 *)(vs[i & 1]) + tid + j * 64 * kPromptWaves;
            h8 v = *at;
            if (drop_non_finite(v)) {
                *at = v;
                odd = true;
            }
        }
        odd = __syncthreads_or(odd);
        if (n0 < wave_max_) {  // else no row of this wave sees the tile
#pragma unroll
            for (int b = 0; b < KT / 32; ++b)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    st[b][e] = n0 + 32 * b + 8 * (e >> 2) + 4 * h + (e & 3) < limit ? st[b][e] : -INFINITY;
            raise();
            weigh();
            add_values(vs[i & 1]);
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
            if (i + 1 < steps) scores(ks[(i + 1) & 1], st);
        }
    }
    sum += other_half(sum);
    if (row >= sp.nq) return;
    const float inv = limit > 0 ? 1.0f / sum : 0.f;
    _Float16 *out = (_Float16 *)a.out.data + (size_t)(sp.q0 + row) * a.out.token_stride + head * a.out.head_stride;
#pragma unroll
    for (int t = 0; t < P::NT; ++t)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            h4 x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = (_Float16)(limit > 0 ? o[t][4 * b + e] * inv : 0.f);
            _Float16 *at = out + 32 * t + 8 * b + 4 * h;
            if (a.out.vec) {
                *(h4 *)at = x;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) at[e] = x[e];
            }
        }
}

template <int D>
hipError_t launch_d(const PromptArgs &a, hipStream_t stream) {
    // every sequence may end in a part tile
    const int tiles = a.q_tokens / kPromptRows + a.sequences;
    attention_prompt_kernel<D><<<dim3((unsigned)tiles * a.q.heads), 64 * kPromptWaves, 0, stream>>>(a, tiles);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_prompt(const PromptArgs &a, hipStream_t stream) {
    if (a.head_dim == 64) return launch_d<64>(a, stream);
    if (a.head_dim == 128) return launch_d<128>(a, stream);
    return launch_d<256>(a, stream);
}

}  // namespace exl3k

// exl3_delta_prompt.hip -- the gated delta rule of long sequences, in chunks of 64 rows.
//
// With G_i the sum of the log decays of a chunk's rows up to i and S the state ahead of it,
//   A_ij = beta_i e^(G_i - G_j) k_i . k_j  (j < i),     T = (1 + A)^-1,
//   U   = T diag(beta) (V - diag(e^G) K S),             (row i of U is the recurrence's u)
//   out = scale (diag(e^G) Q S + P U),                  P_ij = e^(G_i - G_j) q_i . k_j  (j <= i),
//   S  <- e^G_64 S + (diag(e^(G_64 - G)) K)^T U.
// delta_prepare_kernel works out what needs no state for all chunks at once: T by blocks of 16, P, the factors of
// the rows, and lays K and Q out as operands.  delta_scan_kernel walks a sequence's chunks: a workgroup has 16 or
// 32 columns of one head's state in the registers of its waves, 32 rows each, and three exchanges through LDS a chunk.
//
// Bound by the chain from chunk to chunk, three exchanges of about 900 cycles (read, products, write, barrier), in
// which a SIMD has 1500 cycles of instructions of its two waves, and by the preparation's writes.  8192 rows, 16 heads
// of 128: preparation 48 us (0.2 GB, 4.6 TB/s) and walk 159 us, 1.25 us a chunk; 2048 rows 17 and 40 us; 16 sequences
// of 2048 rows 168 and 370 us.  Half the waves carry the state and half make the output, so that the chain has only
// what the next chunk waits for (both on every wave: 400 us in all at 8192 rows).  Where operands lie as lanes want
// them a load is 1 KB of consecutive bytes; 16 rows by 64 bytes a load is four times as slow.
//
// The products run on mfma_f32_16x16x32_f16.  K and Q are fp16 as given (their lengths are factors of rows applied
// afterwards; K's columns have a power of two a row); every other operand x is two fp16 numbers, hi = fp16(x) and
// lo = fp16(x - hi), 22 bits together, after a power of two has taken a bound on its column (or matrix) to 2^15; below
// 2^-29 of that bound they are steps of 2^-40 of it.  Products of two such pairs leave out lo lo.  One fp16 number in
// the state's place would lose what the recurrence in binary32 keeps (2^-11 of S in every chunk).
// (P's one power of two serves rows of any |q|: outputs are fp16, and queries 2^26 apart in length lose none of their bits.)
//
// D leaves lane 16 q + n with column n of rows 4 q + i (i < 4), and B wants rows 8 q + j (j < 8) of column n there.
// So a 32-row operand is two tiles whose rows 4 q + i stand for rows 8 q + i and 8 q + 4 + i: the second
// product's operand is the first one's result, lane for lane.
#include "exl3_delta_step.hpp"

namespace exl3k {

namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

constexpr int kChunk = 64;
// What a chunk and head have in the workspace: the operands of T and P (each six 16 x 32 fragments on and below the
// diagonal, high and low parts, 16 bytes a lane), four factors a row, eight scalars.
constexpr int kFrag = 1024, kFrags = 6;
constexpr int kRowFactors = 2 * kFrags * 2 * kFrag;  // byte offsets
constexpr int kScalars = kRowFactors + 4 * kChunk * 4;
constexpr int kChunkBytes = kScalars + 256;
enum { kRState, kRValue, kUFit, kUBack, kDecay, kWBack, kPBack };  // scalars
// What a chunk and key head have there: the keys as rows (fragment 4 g + t: elements 32 g .., row tile t) and as
// columns (fragment 4 g + 2 k + t: element tile t of 32 g .., rows 32 k ..), the queries as rows (fragment t KD / 32 + g).
constexpr int kKeyFrags = 4;  // a 32 elements, of each
__host__ __device__ constexpr size_t key_bytes(int key_dim) { return (size_t)3 * (key_dim / 32) * kKeyFrags * kFrag; }
// fragment of row tile t (16 rows) and columns 32 s .. 32 s + 31: s <= t / 2
__device__ __forceinline__ int frag_of(int t, int s) { return (t < 2 ? t : 2 * t - 2) + s; }
// The chunk's row that row m of row tile t of K, R, U and T stands for (those of Q, P and out are in their order)
__device__ __forceinline__ int row_of(int t, int m) { return 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3); }

__device__ __forceinline__ f4 mfma16(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// The power of two that takes numbers up to `bound` below 2^15, and its inverse.
struct Fit {
    float to, back;
};
__device__ __forceinline__ Fit fit_of(float bound) {
    int e = __builtin_amdgcn_frexp_expf(bound) - 15;
    e = e < -110 ? -110 : e;
    return {__int_as_float((127 - e) << 23), __int_as_float((127 + e) << 23)};
}

// Two numbers' parts, packed.  In assembly for v_fma_mix_f32 (x - (float)hi in one instruction), and so that hi
// is one value: the compiler fuses the product that made x into one conversion and not into the other, and now
// and then the two are a step apart.
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    float a, b;
    asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(hi) : "v"(x), "v"(y));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(a) : "v"(hi), "v"(x));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(b) : "v"(hi), "v"(y));
    asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(lo) : "v"(a), "v"(b));
}
__device__ __forceinline__ void split4(f4 x, h4 &hi, h4 &lo) {
    u2 a, b;
    uint32_t h, l;
    split2(x[0], x[1], h, l);
    a.x = h, b.x = l;
    split2(x[2], x[3], h, l);
    a.y = h, b.y = l;
    hi = bitcast<h4>(a);
    lo = bitcast<h4>(b);
}
__device__ __forceinline__ void split8(f4 x, f4 y, h8 &hi, h8 &lo) {
    h4 a, b, c, d;
    split4(x, a, b);
    split4(y, c, d);
    hi = (h8){a[0], a[1], a[2], a[3], c[0], c[1], c[2], c[3]};
    lo = (h8){b[0], b[1], b[2], b[3], d[0], d[1], d[2], d[3]};
}

// maximum over lanes l ^ 16, l ^ 32 of numbers that are not negative (as such their bits are in their order)
__device__ __forceinline__ float max_quarters(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    const uint32_t w = max((uint32_t)a[0], (uint32_t)a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return __uint_as_float(max((uint32_t)b[0], (uint32_t)b[1]));
}
__device__ __forceinline__ h2 larger(h2 a, h2 b) { return __builtin_elementwise_max(a, b); }
// over the wave, without LDS
__device__ __forceinline__ float max_lanes(float v) {
    uint32_t w = __float_as_uint(v);
    w = max(w, __float_as_uint(dpp_xor<1>(__uint_as_float(w))));
    w = max(w, __float_as_uint(dpp_xor<2>(__uint_as_float(w))));
    w = max(w, __float_as_uint(dpp_xor<4>(__uint_as_float(w))));
    w = max(w, __float_as_uint(dpp_xor<8>(__uint_as_float(w))));
    return max_quarters(__uint_as_float(w));
}
__device__ __forceinline__ float sum_quarters(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = __int_as_float(a[0]) + __int_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return __int_as_float(b[0]) + __int_as_float(b[1]);
}

// Where 16-byte run c of row r of rows of KD elements in LDS is: 16 rows' runs c lie in all banks, as do a row's runs.
template <int KD>
__device__ __forceinline__ int query_at(int r, int c) {
    return KD == 128 ? r * 128 + 8 * (c ^ (r & 15)) : r * 64 + 8 * (c ^ ((r >> 1) & 7));
}

// Loads stay in their order across this, ahead of the loop as in it: a wait for one is a wait for all that were
// issued before it.
__device__ __forceinline__ void in_order() { asm volatile("" ::: "memory"); }
// What was read from LDS is there: reads that wait for the registers of the products ahead of them come a round trip later.
__device__ __forceinline__ void lds_here() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// The LDS that waves share is complete; loads from memory stay on their way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ------------------------------------------------------------------ what needs no state
constexpr int kRowFloats = kChunk + 4;  // of a matrix in LDS

// One chunk of one value head: wave w has rows 16 w .. 16 w + 15 of the products and column block w of T.
// Workgroups behind those of all tiles and heads take the sequences of fewer than `limit` rows, row by row.
template <int KD>
__global__ __launch_bounds__(256) void delta_prepare_kernel(DeltaArgs a, char *chunks, size_t tiles, int limit, size_t units,
                                                            int slices) {
    constexpr int NK = KD / 32;
    constexpr int kMatrix = kChunk * kRowFloats;
    __shared__ __attribute__((aligned(16))) float lds[3 * kMatrix];  // A, P, T
    __shared__ double sum_lds[kChunk];
    __shared__ float kr_lds[kChunk], qr_lds[kChunk], most_lds[4], l1_lds[4], sum_T_lds[4];
    __shared__ __attribute__((aligned(16))) int shift_lds[kChunk];
    float *const A = lds, *const Pm = lds + kMatrix, *const T = lds + 2 * kMatrix;
    static_assert(kChunk * KD * 2 <= kMatrix * 4, "the keys fit");

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = a.v.heads;
    if (blockIdx.x >= tiles * heads) {
        static_assert(kStepWaves == 4, "a workgroup is a step's");
        const size_t unit = (blockIdx.x - tiles * heads) * kStepWaves + wave;
        if (unit < units) delta_step<KD>(a, unit, slices, limit);
        return;  // the whole workgroup
    }
    const int tile = blockIdx.x / heads, head = blockIdx.x - tile * heads;
    const int m = lane & 15, q = lane >> 4;
    const Tile t = find_tile(a.s, tile, kChunk, lane);
    if (t.s < 0 || t.rows.count < limit) return;  // the whole workgroup
    const int count = min(kChunk, t.rows.count - t.row0);
    if (count <= 0) return;
    const size_t first = (size_t)t.rows.first + t.row0;
    const int kh = head / (heads / a.k.heads);

    // Rows are loaded whole, KD / 8 lanes each, and get into the operands' order through LDS (see output_wave): the
    // keys where T will be, the queries where the wave's own rows of A will be.  Rows beyond the last: zeros, decay 1,
    // beta 0.
    constexpr int L = KD / 8, NR = 16 * L / 64;
    const int row = 16 * wave + m;
    _Float16 *const k_lds = (_Float16 *)T, *const q_lds = (_Float16 *)(A + 16 * wave * kRowFloats);
    // all loads are on their way at once: rows beyond the last are the last one's until they are in registers
    const HeadGates hg = head_gates(a, head);
    Gates gt = load_gates(a, first + min(lane, count - 1), head);
    in_order();
    h8 kx[NR], qx[NR];
#pragma unroll
    for (int j = 0; j < NR; ++j) {
        const int r = 16 * wave + 64 / L * j + lane / L, c = lane % L;
        const size_t at = first + min(r, count - 1);
        kx[j] = load_halves<8>((const _Float16 *)a.k.data + at * a.k.token_stride + kh * a.k.head_stride + 8 * c, a.k.vec);
        qx[j] = load_halves<8>((const _Float16 *)a.q.data + at * a.q.token_stride + kh * a.q.head_stride + 8 * c, a.q.vec);
    }
    in_order();
    // the gates while the rows are on their way
    gt = gates_of(a, hg, gt);
    if (lane >= count) gt = Gates{0.f, 0.f};
    double G = gt.g;  // 64 bits: differences of long sums are the exponents
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(G, d);
        G += lane >= d ? o : 0.0;
    }
    in_order();
#pragma unroll
    for (int j = 0; j < NR; ++j) {
        const int r = 64 / L * j + lane / L, c = lane % L;
        if (16 * wave + r >= count) kx[j] = qx[j] = h8{};
        *(h8 *)(k_lds + query_at<KD>(16 * wave + r, c)) = kx[j];
        *(h8 *)(q_lds + query_at<KD>(r, c)) = qx[j];
    }
    in_order();  // a wave's own rows
    float kk = 0.f, qq = 0.f, k1 = 0.f;
    h8 kf[NK], qf[NK];
#pragma unroll
    for (int s = 0; s < NK; ++s) {
        kf[s] = *(const h8 *)(k_lds + query_at<KD>(row, 4 * s + q));
        qf[s] = *(const h8 *)(q_lds + query_at<KD>(m, 4 * s + q));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = (float)kf[s][j], y = (float)qf[s][j];
            kk = __builtin_fmaf(x, x, kk);
            qq = __builtin_fmaf(y, y, qq);
            k1 += __builtin_fabsf(x);
        }
    }
    kk = sum_quarters(kk);
    qq = sum_quarters(qq);
    k1 = sum_quarters(k1);
    float rk = 1.f, rq = 1.f;
    if (a.eps >= 0.f) {
        rk = inverse_root(kk + a.eps);
        rq = inverse_root(qq + a.eps);
    }
    if (row >= count) rk = rq = 0.f;  // 1 / sqrt(0) where eps is 0
    // The keys' columns are laid out with a power of two a row that takes |k| to 2^14 .. 2^15, and its inverse is in the
    // row's factor of W: one scale serves W's 64 rows, and 1 / |k| there would let the shortest key set it (with a row of
    // zeros and eps = 1e-24 the others' W fell below fp16's steps, and the whole chunk's update was lost).  A row of zeros
    // has none.
    const int shift = kk > 0.f ? 15 - ((__builtin_amdgcn_frexp_expf(kk) + 1) >> 1) : 1000;
    if (wave == 0) sum_lds[lane] = G;
    if (q == 0) {
        kr_lds[row] = rk;
        qr_lds[row] = rq * a.scale;
        shift_lds[row] = shift;
    }
    __syncthreads();

    if (head == kh * (heads / a.k.heads)) {  // one value head of the key head's
        char *const keys = chunks + tiles * heads * (size_t)kChunkBytes + (kh * tiles + tile) * key_bytes(KD);
        h8 *const rows = (h8 *)keys + lane, *const columns = rows + NK * kKeyFrags * 64, *const queries = columns + NK * kKeyFrags * 64;
#pragma unroll
        for (int s = 0; s < NK; ++s) {
            rows[(s * 4 + wave) * 64] = *(const h8 *)(k_lds + query_at<KD>(row_of(wave, m), 4 * s + q));
            queries[(wave * NK + s) * 64] = qf[s];
            // 16 lanes read elements 32 s + 8 c + 4 t .. + 3 (c < 4) of four rows: lane m gets column m of them
            const int k = wave >> 1, t = wave & 1, r = 32 * k + 8 * q + (m >> 2), c = 4 * s + (m & 3);
            const h4 x = bitcast<h4>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(k_lds + query_at<KD>(r, c) + 4 * t)));
            const h4 y = bitcast<h4>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(k_lds + query_at<KD>(r + 4, c) + 4 * t)));
            h8 z;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                z[j] = __builtin_amdgcn_ldexph(j < 4 ? x[j & 3] : y[j & 3], shift_lds[32 * k + 8 * q + j]);
            columns[(s * 4 + wave) * 64] = z;
        }
    }
    // a head's chunks next to each other: the walk over them stays in few pages
    char *const block = chunks + (head * tiles + tile) * kChunkBytes;
    f4 kk_acc[4], qk_acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        kk_acc[j] = qk_acc[j] = (f4){0.f, 0.f, 0.f, 0.f};
        if (j <= wave) {
#pragma unroll
            for (int s = 0; s < NK; ++s) {
                const h8 b = *(const h8 *)(k_lds + query_at<KD>(16 * j + m, 4 * s + q));
                kk_acc[j] = mfma16(kf[s], b, kk_acc[j]);
                qk_acc[j] = mfma16(qf[s], b, qk_acc[j]);
            }
        }
    }
    float p_most = 0.f;
    double Gr[4];
    float brk[4], qr[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = 16 * wave + 4 * q + r;
        Gr[r] = sum_lds[i];
        brk[r] = __shfl(gt.beta, i) * kr_lds[i];
        qr[r] = qr_lds[i];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = 16 * j + m;
        if (j > (wave | 1)) continue;  // above the diagonal's fragments
        if (j > wave) {
#pragma unroll
            for (int r = 0; r < 4; ++r) Pm[(16 * wave + 4 * q + r) * kRowFloats + c] = 0.f;
            continue;
        }
        const double Gc = sum_lds[c];
        const float kc = kr_lds[c];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * wave + 4 * q + r;
            float av = 0.f, pv = 0.f;
            if (i >= c) {
                // a row's factor meets the product ahead of the other row's: 1 / |k| of two rows of zeros may be 2^74 each
                const float fall = decay_of((float)(Gr[r] - Gc)) * kc;
                pv = qr[r] * qk_acc[j][r] * fall;
                if (i > c) av = brk[r] * kk_acc[j][r] * fall;
            }
            A[i * kRowFloats + c] = av;
            Pm[i * kRowFloats + c] = pv;
            p_most = fmaxf(p_most, __builtin_fabsf(pv));
        }
    }
    p_most = max_lanes(p_most);
    if (lane == 0) most_lds[wave] = p_most;
    // row factors and scalars, by the wave that has the rows' k1: each wave its 16, wave 0 all
    const float beta_row = __shfl(gt.beta, row);
    const float since = decay_of((float)__shfl(G, row)) * rk;
    const float l1 = max_lanes(__builtin_fabsf(beta_row * since) * k1);
    if (lane == 0) l1_lds[wave] = l1;
    const double G_end = __shfl(G, 63);
    __syncthreads();

    // the inverse of the diagonal block, column m of it in every lane of four: forward substitution
    float t_col[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float v = i == m ? 1.f : 0.f;
        const float *const A_row = A + (16 * wave + i) * kRowFloats + 16 * wave;
#pragma unroll
        for (int j = 0; j < i; ++j) v = __builtin_fmaf(-A_row[j], t_col[j], v);
        t_col[i] = v;
        if (q == 0) T[(16 * wave + i) * kRowFloats + 16 * wave + m] = v;
    }
    float t_most = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t_most = fmaxf(t_most, __builtin_fabsf(t_col[i]));
    __syncthreads();
    // T_ij = -T_ii sum_{j <= l < i} A_il T_lj, column block j = wave; step r of a product takes its rows
    // 4 q + r, which is where D left them
    f4 T_col[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) T_col[0][r] = T[(16 * wave + 4 * q + r) * kRowFloats + 16 * wave + m];
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        T_col[i] = (f4){0.f, 0.f, 0.f, 0.f};
        const int bi = wave + i;
        if (bi < 4) {
            f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int l = 0; l < i; ++l) {
                const f4 x = *(const f4 *)(A + (16 * bi + m) * kRowFloats + 16 * (wave + l) + 4 * q);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r], T_col[l][r], acc, 0, 0, 0);
            }
            const f4 x = *(const f4 *)(T + (16 * bi + m) * kRowFloats + 16 * bi + 4 * q);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                T_col[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(-x[r], acc[r], T_col[i], 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r) t_most = fmaxf(t_most, __builtin_fabsf(T_col[i][r]));
        }
    }
    const float p_top = fmaxf(fmaxf(most_lds[0], most_lds[1]), fmaxf(most_lds[2], most_lds[3]));
    __syncthreads();  // the diagonal blocks and most_lds have been read
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        const int bi = (wave + i) & 3;  // below the diagonal, or zeros above it
#pragma unroll
        for (int r = 0; r < 4; ++r)
            T[(16 * bi + 4 * q + r) * kRowFloats + 16 * wave + m] = wave + i < 4 ? T_col[i][r] : 0.f;
    }
    t_most = max_lanes(t_most);
    if (lane == 0) most_lds[wave] = t_most;
    __syncthreads();
    const float t_top = fmaxf(fmaxf(most_lds[0], most_lds[1]), fmaxf(most_lds[2], most_lds[3]));
    const Fit tf = fit_of(t_top), pf = fit_of(p_top);

    // the fragments of row tile `wave`
    float t_sum = 0.f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if (s > wave >> 1) break;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const float *const from =
                (which ? Pm + row * kRowFloats : T + row_of(wave, m) * kRowFloats) + 32 * s + 8 * q;
            const float to = which ? pf.to : tf.to;
            h8 hi, lo;
            split8(*(const f4 *)from * to, *(const f4 *)(from + 4) * to, hi, lo);
            if (!which) {
#pragma unroll
                for (int j = 0; j < 8; ++j) t_sum += __builtin_fabsf(from[j]);
            }
            h8 *const at = (h8 *)(block + ((which * kFrags + frag_of(wave, s)) * 2) * kFrag) + lane;
            at[0] = hi;
            at[64] = lo;
        }
    }
    t_sum = max_lanes(sum_quarters(t_sum));
    if (lane == 0) sum_T_lds[wave] = t_sum;
    __syncthreads();
    if (wave == 0) {  // lane = row
        const float r = kr_lds[lane], e = decay_of((float)G);
        const float until = __builtin_amdgcn_ldexpf(decay_of((float)(G_end - G)) * r, -shift_lds[lane]);
        int e_w = __builtin_amdgcn_frexp_expf(max_lanes(__builtin_fabsf(until)));
        e_w = e_w < -110 ? -110 : e_w;
        float *const f = (float *)(block + kRowFactors);
        f[lane] = e * r;
        f[kChunk + lane] = e * qr_lds[lane];
        f[2 * kChunk + lane] = gt.beta;
        f[3 * kChunk + lane] = __builtin_amdgcn_ldexpf(until, -e_w);
        const float beta_most = max_lanes(__builtin_fabsf(gt.beta));
        if (lane == 0) {
            float *const s = (float *)(block + kScalars);
            s[kDecay] = decay_of((float)G_end);
            // |U| <= (largest row sum of T) |R|: another power of two keeps U where R was
            const int e_u = __builtin_amdgcn_frexp_expf(
                fmaxf(fmaxf(sum_T_lds[0], sum_T_lds[1]), fmaxf(sum_T_lds[2], sum_T_lds[3])));
            s[kUFit] = __builtin_amdgcn_ldexpf(tf.back, -e_u);
            s[kUBack] = __builtin_amdgcn_ldexpf(1.f, e_u);
            s[kPBack] = pf.back;
            s[kWBack] = __builtin_amdgcn_ldexpf(1.f, e_w);
            s[kRState] = fmaxf(fmaxf(l1_lds[0], l1_lds[1]), fmaxf(l1_lds[2], l1_lds[3]));
            s[kRValue] = beta_most;
            s[7] = 0.f;  // loaded along
        }
    }
}

// ------------------------------------------------------------------ the walk over the chunks
// chunks of the sequences ahead of s
__device__ __forceinline__ size_t tiles_before(const Sequences &p, int s, int lane) {
    if (!p.starts) {
        const int n = p.tokens / p.sequences;
        return (size_t)s * (n > kChunk ? (n + kChunk - 1) / kChunk : 1);
    }
    unsigned long long sum = 0;
    for (int i = lane; i < s; i += 64) {
        const int n = rows_of(p, i).count;
        sum += n > kChunk ? (n + kChunk - 1) / kChunk : 1;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    return sum;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ size_t uniform(size_t v) {
    return (uint32_t)uniform((int)(uint32_t)v) | (size_t)(uint32_t)uniform((int)(uint32_t)(v >> 32)) << 32;
}

// A workgroup has columns 16 NC slice .. of one head's state, NC tiles of them, and two kinds of waves, KD / 32 of
// each.  State wave w has rows 32 w .. 32 w + 31 of the state, as two tiles, and TT of the chunk's four row tiles of R
// and U: what the next chunk waits for.  Output wave w has Q S, P U and out of TT row tiles, and the first two (all
// where NC is 2) bring V into LDS.  Everything else is read as operands, straight from the workspace.  VEC: 16 bytes of
// a row of v and out are one access.
//
// LDS, by the barrier (1 to 3 of a chunk) that its writes are ahead of and the one that its reads are ahead of:
// s, back, ks: 1, 2;  v: 3 of the chunk before, 2;  v_top: 1, 2;  r, u_back: 2, 3;  u, w: 3, 1 of the next.  A buffer is
// written again only past the barrier that its reads are ahead of.  o is a wave's own.
template <int KD, int NC>
struct ScanLds {
    static constexpr int NW = KD / 32;
    static constexpr int kValueWaves = NC == 1 ? 2 : NW;  // output waves that bring V
    h8 s[NC][NW][2][64];              // the state's operand: 32 rows, high and low
    f4 ks[NC][NW][4][64];             // K S of those rows alone, the chunk's row tiles
    h8 r[NC][2][2][64];               // R's, 32 rows each
    h8 u[NC][2][2][64], w[NC][2][2][64];
    _Float16 v[kChunk][16 * NC], o[kChunk][16 * NC];
    float back[NC][NW][16], u_back[NC][16], v_top[kValueWaves];
};

struct ScanPlace {
    Rows rows;
    const char *block, *keys;  // the first chunk's parts of the workspace
    int n_chunks, head, slice, slot_in, slot_out;
};

// A sequence's rows, a chunk of them at a time, as a buffer: what is beyond the last row reads as zero and is not written.
typedef __amdgpu_buffer_rsrc_t Buffer;
struct ChunkRows {
    char *base;      // the chunk's first row
    uint32_t row;    // bytes from a row to the next
    int left, width; // rows of the sequence from the chunk's on, bytes of a row that are used
    __device__ __forceinline__ ChunkRows(const Heads &h, const ScanPlace &p, int head, int at, int elements) {
        base = (char *)((_Float16 *)h.data + p.rows.first * h.token_stride + head * h.head_stride + at);
        row = (uint32_t)(2 * h.token_stride);
        left = p.rows.count;
        width = 2 * elements;
    }
    __device__ __forceinline__ Buffer buffer() const {
        const int n = min(left, kChunk);
        return __builtin_amdgcn_make_buffer_rsrc(base, 0, n > 0 ? (n - 1) * row + width : 0, 0x00020000);
    }
    __device__ __forceinline__ void step() {
        base += (size_t)row * kChunk;
        left -= kChunk;
    }
};
template <bool VEC>
__device__ __forceinline__ h8 load_run(Buffer b, uint32_t at) {
    if constexpr (VEC) {
        return bitcast<h8>(__builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0));
    } else {
        h8 t;
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = bitcast<_Float16>(__builtin_amdgcn_raw_buffer_load_b16(b, at + 2 * e, 0, 0));
        return t;
    }
}

// A part of the workspace that is read chunk by chunk; behind the last chunk it is the last one's again.
struct Part {
    const char *at;
    size_t distance;
    int left;
    __device__ __forceinline__ Part(const char *first, size_t step, int n) : at(first), distance(step), left(n) {}
    __device__ __forceinline__ void step() { at += --left > 0 ? distance : 0; }
};
// T's or P's fragments of a wave's row tiles: G of them each
template <int TT, int G>
__device__ __forceinline__ void load_matrix(const char *from, int wave, int lane, h8 (&to)[TT][G][2]) {
    const h8 *const f = (const h8 *)from + lane;
#pragma unroll
    for (int tt = 0; tt < TT; ++tt)
#pragma unroll
        for (int g = 0; g < G; ++g) {
            to[tt][g][0] = f[frag_of(wave * TT + tt, g) * 128];
            to[tt][g][1] = f[frag_of(wave * TT + tt, g) * 128 + 64];
        }
}
// A row tile of T or P times R or U (b's first 32 rows, or all 64)
template <int G>
__device__ __forceinline__ void read_pairs(const h8 (&b)[2][2][64], int lane, h8 (&to)[G][2]) {
#pragma unroll
    for (int g = 0; g < G; ++g) to[g][0] = b[g][0][lane], to[g][1] = b[g][1][lane];
}
template <int G>
__device__ __forceinline__ f4 lower_product(const h8 (&m)[G][2], const h8 (&b)[G][2]) {
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    f4 x = zero, y = zero, z = zero;
#pragma unroll
    for (int g = 0; g < G; ++g) {
        x = mfma16(m[g][0], b[g][0], x);
        y = mfma16(m[g][0], b[g][1], y);
        z = mfma16(m[g][1], b[g][0], z);
    }
    return x + (y + z);
}
template <typename L>
__device__ __forceinline__ void put_quarter(L &lds, int t, int lane, f4 x) {
    h4 hi, lo;
    split4(x, hi, lo);
    *((h4 *)&lds[t >> 1][0][lane] + (t & 1)) = hi;
    *((h4 *)&lds[t >> 1][1][lane] + (t & 1)) = lo;
}
// K S or Q S of a row tile
template <int NW>
__device__ __forceinline__ f4 state_product(const h8 (&rows)[NW], const h8 (&hi)[NW], const h8 (&lo)[NW], const float (&back)[NW]) {
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    f4 x[NW], y;
#pragma unroll
    for (int g = 0; g < NW; ++g) x[g] = mfma16(rows[g], hi[g], zero);
#pragma unroll
    for (int g = 0; g < NW; ++g) x[g] = mfma16(rows[g], lo[g], x[g]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        y[i] = x[0][i] * back[0];
#pragma unroll
        for (int g = 1; g < NW; ++g) y[i] = __builtin_fmaf(x[g][i], back[g], y[i]);
    }
    return y;
}

// UPPER: the wave's row tiles are those of rows 32 .. 63, with two fragments of T or P each
template <int KD, int NC, bool UPPER>
__device__ __forceinline__ void state_wave(const DeltaArgs &a, const ScanPlace &p, ScanLds<KD, NC> &lds, int wave, int lane) {
    constexpr int NW = KD / 32, TT = 4 / NW, G = UPPER ? 2 : 1;
    const int m = lane & 15, q = lane >> 4;
    const size_t state_size = (size_t)a.v.heads * KD * a.value_dim;
    const size_t state_at = ((size_t)p.head * KD + 32 * wave + 8 * q) * a.value_dim + 16 * NC * p.slice + m;
    f4 S[NC][2];
    const float start = p.slot_in == kBadState ? __builtin_nanf("") : 0.f;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                S[n][t][i] = p.slot_in >= 0
                                 ? a.states[p.slot_in * state_size + state_at + (size_t)(4 * t + i) * a.value_dim + 16 * n]
                                 : start;
#pragma unroll
    for (int n = 0; n < NC; ++n)  // waited for here: in the loop it would be a wait for all loads
        asm volatile("" : "+v"(S[n][0]), "+v"(S[n][1]));

    // the keys' 32 elements of the wave, as rows of the chunk's tiles and as columns
    h8 kf[4], kt[2][2], tf[TT][G][2];
    f4 fk[TT], fb[TT], fu[TT];
    float sc[8], next_sc[8];  // through registers of the lanes: a scalar load would be waited for with LDS
    Part rows(p.keys + wave * 4 * kFrag, key_bytes(KD), p.n_chunks), factors(p.block + kRowFactors, kChunkBytes, p.n_chunks),
        t_part(p.block, kChunkBytes, p.n_chunks), columns(p.keys + (NW + wave) * 4 * kFrag, key_bytes(KD), p.n_chunks);
    auto load_rows = [&]() {
#pragma unroll
        for (int t = 0; t < 4; ++t) kf[t] = ((const h8 *)rows.at)[64 * t + lane];
        rows.step();
        in_order();
    };
    auto load_factors = [&]() {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const int r4 = row_of(wave * TT + tt, 4 * q) / 4;
            fk[tt] = ((const f4 *)factors.at)[r4];
            fb[tt] = ((const f4 *)factors.at)[2 * kChunk / 4 + r4];
            fu[tt] = ((const f4 *)factors.at)[3 * kChunk / 4 + r4];
        }
        const f4 x = ((const f4 *)(factors.at + kScalars - kRowFactors))[0], y = ((const f4 *)(factors.at + kScalars - kRowFactors))[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) next_sc[i] = x[i], next_sc[4 + i] = y[i];
        factors.step();
        in_order();
    };
    auto load_t = [&]() {
        load_matrix<TT, G>(t_part.at, wave, lane, tf);
        t_part.step();
        in_order();
    };
    auto load_columns = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i) kt[i >> 1][i & 1] = ((const h8 *)columns.at)[64 * i + lane];
        columns.step();
        in_order();
    };
    if (p.n_chunks) {
        in_order();
        load_rows();
        load_factors();
        load_t();
        lds_barrier();
    }
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < p.n_chunks; ++c) {
#pragma unroll
        for (int i = 0; i < 7; ++i) sc[i] = next_sc[i];
        // the state as an operand, each wave's rows by their own power of two a column
        h8 hi[NC], lo[NC];
        float s_fit[NC];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            float top = 0.f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, __builtin_fabsf(S[n][t][i]));
            const Fit sf = fit_of(max_quarters(top));
            split8(S[n][0] * sf.to, S[n][1] * sf.to, hi[n], lo[n]);
            s_fit[n] = sf.back;
        }
        f4 x[NC][4];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
#pragma unroll
            for (int t = 0; t < 4; ++t) x[n][t] = mfma16(kf[t], hi[n], zero);
#pragma unroll
            for (int t = 0; t < 4; ++t) x[n][t] = mfma16(kf[t], lo[n], x[n][t]);
        }
        in_order();
        load_columns();
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            lds.s[n][wave][0][lane] = hi[n];
            lds.s[n][wave][1][lane] = lo[n];
            if (q == 0) lds.back[n][wave][m] = s_fit[n];
        }
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int t = 0; t < 4; ++t) lds.ks[n][wave][t][lane] = x[n][t];
        lds_barrier();  // 1

        // R = beta (V - e^G K S), |R| <= r_value |V| + r_state |S|
        f4 ks[NC][TT][NW];
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                for (int g = 0; g < NW; ++g) ks[n][tt][g] = lds.ks[n][g][wave * TT + tt][lane];
        in_order();  // loads are issued while LDS answers
        load_rows();
        float v_top = lds.v_top[0];
#pragma unroll
        for (int i = 1; i < ScanLds<KD, NC>::kValueWaves; ++i) v_top = fmaxf(v_top, lds.v_top[i]);
        float u_back[NC];
        f4 w_fit[TT];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            float back[NW], s_back = 0.f;
#pragma unroll
            for (int g = 0; g < NW; ++g) {
                back[g] = lds.back[n][g][m];
                s_back = fmaxf(s_back, back[g]);
            }
            const Fit rf = fit_of(__builtin_fmaf(sc[kRState] * 32768.f, s_back, sc[kRValue] * v_top));
            u_back[n] = rf.back * sc[kUBack];
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                const int t = wave * TT + tt;
                // 16 lanes read four rows of V: lane m gets column m of them
                const h4 v = bitcast<h4>(__builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds_s4 *)&lds.v[row_of(t, 4 * q) + (m >> 2)][16 * n + 4 * (m & 3)]));
                f4 y, r;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    y[i] = ks[n][tt][0][i] * back[0];
#pragma unroll
                    for (int g = 1; g < NW; ++g) y[i] = __builtin_fmaf(ks[n][tt][g][i], back[g], y[i]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = fb[tt][i] * rf.to * __builtin_fmaf(-fk[tt][i], y[i], (float)v[i]);
                put_quarter(lds.r[n], t, lane, r);
            }
            if (wave == 0 && q == 0) lds.u_back[n][m] = u_back[n];
        }
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) w_fit[tt] = fu[tt];
        lds_barrier();  // 2

        // U = T R, and W = e^(G_64 - G) U for the state
        h8 r[NC][G][2];
#pragma unroll
        for (int n = 0; n < NC; ++n) read_pairs<G>(lds.r[n], lane, r[n]);
        in_order();
        load_factors();
        lds_here();
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                const f4 u = lower_product<G>(tf[tt], r[n]) * sc[kUFit];
                put_quarter(lds.w[n], wave * TT + tt, lane, u * w_fit[tt]);
                put_quarter(lds.u[n], wave * TT + tt, lane, u);
            }
        in_order();
        load_t();
        lds_barrier();  // 3

        // S <- e^G_64 S + K^T W
        h8 w[NC][2][2];
#pragma unroll
        for (int n = 0; n < NC; ++n) read_pairs<2>(lds.w[n], lane, w[n]);
        lds_here();
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            f4 acc[2] = {zero, zero}, acc_lo[2] = {zero, zero};
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    acc[t] = mfma16(kt[g][t], w[n][g][0], acc[t]);
                    acc_lo[t] = mfma16(kt[g][t], w[n][g][1], acc_lo[t]);
                }
            const float s_more = u_back[n] * sc[kWBack];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    S[n][t][i] = __builtin_fmaf(acc[t][i] + acc_lo[t][i], s_more, sc[kDecay] * S[n][t][i]);
        }
    }
    if (p.slot_out >= 0) {
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    a.states[p.slot_out * state_size + state_at + (size_t)(4 * t + i) * a.value_dim + 16 * n] = S[n][t][i];
    }
}

template <int KD, int NC, bool VEC, bool UPPER>
__device__ __forceinline__ void output_wave(const DeltaArgs &a, const ScanPlace &p, ScanLds<KD, NC> &lds, int wave, int lane) {
    constexpr int NW = KD / 32, TT = 4 / NW, G = UPPER ? 2 : 1;
    // known when compiled, so that the compiler can count the loads that are on their way
    constexpr bool kValues = NC == 2 || !UPPER || NW == 2;
    constexpr int PR = 2 * NC, VL = NC * 2 / ScanLds<KD, NC>::kValueWaves;  // 16-byte pieces a row, loads of V a lane
    if (!p.n_chunks) return;
    const int m = lane & 15, q = lane >> 4;
    ChunkRows o_rows(a.out, p, p.head, 16 * NC * p.slice, 16 * NC), v_rows(a.v, p, p.head, 16 * NC * p.slice, 16 * NC);
    // 16 rows of a tile, PR lanes each.  The store is not left out by any lane or chunk (a place beyond the buffer is not
    // written): where the compiler cannot count it, it waits for it together with the loads that it knows.
    uint32_t o_at[TT];
#pragma unroll
    for (int tt = 0; tt < TT; ++tt)
        o_at[tt] = lane < 16 * PR ? (uint32_t)(16 * (wave * TT + tt) + lane / PR) * o_rows.row + 16 * (lane % PR) : 0xfffffff0u;
    // values: 64 / PR rows a load
    int v_row[VL];
    uint32_t v_at[VL];
#pragma unroll
    for (int j = 0; j < VL; ++j) {
        v_row[j] = 64 / PR * (wave * VL + j) + lane / PR;
        v_at[j] = (uint32_t)v_row[j] * v_rows.row + 16 * (lane % PR);
    }

    h8 qf[TT][NW], pf[TT][G][2], vr[VL];
    f4 fq[TT], pu[NC][TT] = {}, qs[NC][TT] = {};
    float o_back[NC] = {}, p_back;
    Part queries(p.keys + (2 * NW * 4 + wave * TT * NW) * kFrag, key_bytes(KD), p.n_chunks),
        factors(p.block + kRowFactors, kChunkBytes, p.n_chunks), p_part(p.block + kFrags * 2 * kFrag, kChunkBytes, p.n_chunks),
        scalar(p.block + kScalars + 4 * kPBack, kChunkBytes, p.n_chunks);
    auto load_p_back = [&]() {
        p_back = *(const float *)scalar.at;
        scalar.step();
        in_order();
    };
    auto load_q = [&]() {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
#pragma unroll
            for (int g = 0; g < NW; ++g) qf[tt][g] = ((const h8 *)queries.at)[64 * (tt * NW + g) + lane];
            fq[tt] = ((const f4 *)factors.at)[kChunk / 4 + 4 * (wave * TT + tt) + q];
        }
        queries.step();
        factors.step();
        in_order();
    };
    auto load_p = [&]() {
        load_matrix<TT, G>(p_part.at, wave, lane, pf);
        p_part.step();
        in_order();
    };
    auto load_v = [&]() {  // zeros behind the last chunk
        if (kValues) {
#pragma unroll
            for (int j = 0; j < VL; ++j) vr[j] = load_run<VEC>(v_rows.buffer(), v_at[j]);
        }
        v_rows.step();
        in_order();
    };
    h2 top = {};
    auto put_v = [&]() {
        if (kValues) {
#pragma unroll
            for (int j = 0; j < VL; ++j) {
                *(h8 *)&lds.v[v_row[j]][8 * (lane % PR)] = vr[j];
                const u4 x = bitcast<u4>(vr[j]) & 0x7fff7fffu;
                const h2 y = larger(larger(bitcast<h2>(x.x), bitcast<h2>(x.y)), larger(bitcast<h2>(x.z), bitcast<h2>(x.w)));
                top = j ? larger(top, y) : y;
            }
        }
    };
    // the largest |V| of the wave's rows; infinities and NaN count as fp16's largest, for the other columns
    auto put_top = [&]() {
        if (kValues) {
            const float x = fminf(max_lanes(fmaxf((float)top[0], (float)top[1])), 65504.f);
            if (lane == 0) lds.v_top[wave] = x;
        }
    };
    auto put_out = [&](Buffer b) {  // e^G Q S + P U
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const int t = wave * TT + tt;
#pragma unroll
            for (int n = 0; n < NC; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    lds.o[16 * t + 4 * q + i][16 * n + m] = (_Float16)__builtin_fmaf(pu[n][tt][i], o_back[n], qs[n][tt][i]);
            const h8 o = *(const h8 *)&lds.o[16 * t + (lane / PR & 15)][8 * (lane % PR)];
            if constexpr (VEC) {
                __builtin_amdgcn_raw_buffer_store_b128(bitcast<u4>(o), b, o_at[tt], 0, 0);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    __builtin_amdgcn_raw_buffer_store_b16(bitcast<uint16_t>((_Float16)o[e]), b, o_at[tt] + 2 * e, 0, 0);
            }
        }
        in_order();
    };
    load_v();
    put_v();
    put_top();
    in_order();
    load_q();
    load_v();
    load_p_back();
    load_p();
    lds_barrier();
    Buffer before = __builtin_amdgcn_make_buffer_rsrc(o_rows.base, 0, 0, 0x00020000);  // nothing ahead of the first chunk
    for (int c = 0; c < p.n_chunks; ++c) {
        lds_barrier();  // 1
        f4 qs_now[NC][TT];
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            h8 s_hi[NW], s_lo[NW];
            float back[NW];
#pragma unroll
            for (int g = 0; g < NW; ++g) {
                s_hi[g] = lds.s[n][g][0][lane];
                s_lo[g] = lds.s[n][g][1][lane];
                back[g] = lds.back[n][g][m];
            }
            lds_here();
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) qs_now[n][tt] = state_product<NW>(qf[tt], s_hi, s_lo, back) * fq[tt];
        }
        in_order();
        load_q();
        lds_barrier();  // 2
        put_out(before);
        put_v();
        in_order();
        load_v();
#pragma unroll
        for (int n = 0; n < NC; ++n) o_back[n] = lds.u_back[n][m] * p_back;
        in_order();
        load_p_back();
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) qs[n][tt] = qs_now[n][tt];
        before = o_rows.buffer();
        o_rows.step();
        lds_barrier();  // 3
        h8 u[NC][G][2];
#pragma unroll
        for (int n = 0; n < NC; ++n) read_pairs<G>(lds.u[n], lane, u[n]);
        lds_here();
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) pu[n][tt] = lower_product<G>(pf[tt], u[n]);
        in_order();
        load_p();
        put_top();
    }
    put_out(before);
}

template <int KD, int NC, bool VEC>
__global__ __launch_bounds__(4 * KD) void delta_scan_kernel(DeltaArgs a, const char *chunks, size_t tiles, int units,
                                                            int slices, int limit) {
    constexpr int NW = KD / 32;
    __shared__ __attribute__((aligned(16))) ScanLds<KD, NC> lds;
    // the slices of a head on one XCD, whose L2 then holds what they share
    const int id = blockIdx.x, at_xcd = id >> 3;
    const int unit = at_xcd / slices * 8 + (id & 7);
    if (unit >= units) return;
    const int heads = a.v.heads, s = unit / heads;
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
    ScanPlace p;
    p.slice = at_xcd % slices;
    p.head = unit - s * heads;
    const int kh = p.head / (heads / a.k.heads);
    const Rows rows = rows_of(a.s, s);
    p.rows = {uniform(rows.first), uniform(rows.count)};
    if (p.rows.count < limit) return;  // the whole workgroup
    p.slot_in = uniform(slot_in(a.s, s));
    p.slot_out = uniform(slot_out(a.s, s));
    const size_t tile0 = uniform(tiles_before(a.s, s, lane));
    // starts that overlap have more chunks than the workspace holds: those are left out
    p.n_chunks = (int)min((size_t)(p.rows.count + kChunk - 1) / kChunk, tiles - min(tiles, tile0));
    p.block = chunks + (p.head * tiles + tile0) * kChunkBytes;
    p.keys = chunks + heads * tiles * kChunkBytes + (kh * tiles + tile0) * key_bytes(KD);
    if (wave < NW / 2) state_wave<KD, NC, false>(a, p, lds, wave, lane);
    else if (wave < NW) state_wave<KD, NC, true>(a, p, lds, wave, lane);
    else if (wave < NW + NW / 2) output_wave<KD, NC, VEC, false>(a, p, lds, wave - NW, lane);
    else output_wave<KD, NC, VEC, true>(a, p, lds, wave - NW, lane);
}

// Parts of 16 columns of all sequences and heads from which on a workgroup takes 32 of them: their operands are
// loaded once and the longer chain is hidden by nothing, but the card is full either way.  16 heads of 128, sequences of
// 2048 rows, walk alone, 16 and 32 columns: 2 sequences (256 parts) 41 and 70 us, 4: 87 and 79, 6: 171 and 173, 8: 219 and
// 182, 16: 423 and 354 us.  16 heads with keys of 64, where the wide kernel has one workgroup a CU and the narrow one two:
// values of 128, 4 sequences (512 parts) 66 and 74 us, 6: 118 and 149, 8: 163 and 161, 16: 325 and 324; values of 64, 16
// sequences (1024 parts) 196 and 174 us.
constexpr size_t kWideParts = 1024;

template <int KD, int NC>
void launch_scan(const DeltaArgs &a, const char *chunks, size_t tiles, int limit, hipStream_t stream) {
    const int units = a.s.sequences * a.v.heads, slices = a.value_dim / (16 * NC);
    const dim3 blocks((unsigned)((units + 7) / 8 * 8 * slices));
    if (a.v.vec && a.out.vec)
        delta_scan_kernel<KD, NC, true><<<blocks, dim3(4 * KD), 0, stream>>>(a, chunks, tiles, units, slices, limit);
    else
        delta_scan_kernel<KD, NC, false><<<blocks, dim3(4 * KD), 0, stream>>>(a, chunks, tiles, units, slices, limit);
}

template <int KD>
hipError_t launch_kd(const DeltaArgs &a, char *chunks, hipStream_t stream) {
    const size_t tiles = tile_count(a.s, kChunk), heads = a.v.heads, slices = a.value_dim / 16;
    // sequences of one length are all long ones; one alone goes in chunks whatever its length
    const int limit = a.s.starts && a.s.sequences > 1 ? (int)kDeltaShortRows : 0;
    const size_t parts = a.s.sequences * heads * slices, steps = limit ? parts : 0;
    delta_prepare_kernel<KD><<<dim3((unsigned)(tiles * heads + (steps + kStepWaves - 1) / kStepWaves)), dim3(256), 0, stream>>>(
        a, chunks, tiles, limit, steps, (int)slices);
    if (parts >= kWideParts && slices % 2 == 0) launch_scan<KD, 2>(a, chunks, tiles, limit, stream);
    else launch_scan<KD, 1>(a, chunks, tiles, limit, stream);
    return hipGetLastError();
}

}  // namespace

bool delta_prompt_serves(const DeltaArgs &a) {
    const size_t most = (size_t)1 << 24, parts = (size_t)a.s.sequences * a.v.heads * (a.value_dim / 16);
    const size_t rows = parts < kDeltaManyParts ? kDeltaPromptRows : kDeltaPromptRowsOfMany;
    return (a.s.starts || a.s.tokens >= rows * a.s.sequences) && a.v.token_stride <= most && a.out.token_stride <= most;
}

size_t delta_prompt_bytes(size_t heads, int key_dim, size_t sequences, size_t tokens) {
    if (tokens < kDeltaPromptRows || tokens < kDeltaMixedRows * sequences) return 0;
    // as many key heads as value heads
    return kSharedPrefixBytes + (tokens / kChunk + sequences) * heads * (kChunkBytes + key_bytes(key_dim));
}

hipError_t launch_delta_prompt(const DeltaArgs &a, void *workspace, hipStream_t stream) {
    char *const chunks = (char *)workspace + kSharedPrefixBytes;
    return a.key_dim == 64 ? launch_kd<64>(a, chunks, stream) : launch_kd<128>(a, chunks, stream);
}

}  // namespace exl3k

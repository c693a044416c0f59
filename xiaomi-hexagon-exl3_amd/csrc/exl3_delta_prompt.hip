// exl3_delta_prompt.hip -- the gated delta rule of long sequences, in chunks of 64 rows.
//
// With G_i the sum of the log decays of a chunk's rows up to i and S the state ahead of it,
//   A_ij = beta_i e^(G_i - G_j) k_i . k_j  (j < i),     T = (1 + A)^-1,
//   U   = T diag(beta) (V - diag(e^G) K S),             (row i of U is the recurrence's u)
//   out = scale (diag(e^G) Q S + P U),                  P_ij = e^(G_i - G_j) q_i . k_j  (j <= i),
//   S  <- e^G_64 S + (diag(e^(G_64 - G)) K)^T U.
// delta_prepare_kernel works out what needs no state for all chunks at once: T by blocks of 16, P, and the
// factors of the rows.  delta_scan_kernel walks a sequence's chunks: a workgroup has 16 columns of one head's state
// in the registers of its waves, 32 rows each, and three exchanges through LDS a chunk.
//
// The products run on mfma_f32_16x16x32_f16.  K and Q are fp16 as given (their lengths are factors of rows
// applied afterwards); every other operand x is two fp16 numbers, hi = fp16(x) and lo = fp16(x - hi), 22 bits
// together, after a power of two has taken a bound on its column (or matrix) to 2^15; below 2^-29 of that bound
// they are steps of 2^-40 of it.  Products of two such pairs leave out lo lo.  One fp16 number in the state's place would lose what the recurrence in binary32 keeps
// (2^-11 of S in every chunk).
//
// D leaves lane 16 q + n with column n of rows 4 q + i (i < 4), and B wants rows 8 q + j (j < 8) of column n there.
// So a 32-row operand is two tiles whose rows 4 q + i stand for rows 8 q + i and 8 q + 4 + i: the second
// product's operand is the first one's result, lane for lane.
#include "exl3_delta_gates.hpp"
#include "exl3_head_rows.hpp"

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
enum { kDecay, kUFit, kUBack, kPBack, kWFit, kWBack, kRState, kRValue };  // scalars
// fragment of row tile t (16 rows) and columns 32 s .. 32 s + 31: s <= t / 2
__device__ __forceinline__ int frag_of(int t, int s) { return (t < 2 ? t : 2 * t - 2) + s; }
// the chunk's row that row m of row tile t stands for
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

// A number's parts.  x is kept opaque: fused into the conversion, the product that made it is rounded once for hi and
// twice for the hi that lo is the rest of, and now and then they are a step apart.
__device__ __forceinline__ void split(float x, _Float16 &hi, _Float16 &lo) {
    asm("" : "+v"(x));
    hi = (_Float16)x;
    lo = (_Float16)(x - (float)hi);
}

// maximum over lanes l ^ 16, l ^ 32
__device__ __forceinline__ float max_quarters(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = fmaxf(__int_as_float(a[0]), __int_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return fmaxf(__int_as_float(b[0]), __int_as_float(b[1]));
}
__device__ __forceinline__ float sum_quarters(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = __int_as_float(a[0]) + __int_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    return __int_as_float(b[0]) + __int_as_float(b[1]);
}

__device__ __forceinline__ h8 load_h8(const _Float16 *p, int vec) {
    if (vec) return *(const h8 *)p;
    h8 t;
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = p[e];
    return t;
}

// The LDS that waves share is complete; loads from memory stay on their way.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ------------------------------------------------------------------ what needs no state
constexpr int kRowFloats = kChunk + 4;  // of a matrix in LDS

// One chunk of one value head: wave w has rows 16 w .. 16 w + 15 of the products and column block w of T.
template <int KD>
__global__ __launch_bounds__(256) void delta_prepare_kernel(DeltaArgs a, char *chunks) {
    constexpr int NK = KD / 32;
    constexpr int kMatrix = kChunk * kRowFloats;
    __shared__ __attribute__((aligned(16))) float lds[3 * kMatrix];  // A, P, T
    __shared__ double sum_lds[kChunk];
    __shared__ float kr_lds[kChunk], qr_lds[kChunk], most_lds[4], l1_lds[4], sum_T_lds[4];
    float *const A = lds, *const Pm = lds + kMatrix, *const T = lds + 2 * kMatrix;
    h8 *const kf_lds = (h8 *)T;  // the keys' fragments, until T takes their place
    static_assert(4 * NK * kFrag <= kMatrix * 4, "the keys fit");

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = a.v.heads, tile = blockIdx.x / heads, head = blockIdx.x - tile * heads;
    const int m = lane & 15, q = lane >> 4;
    const Tile t = find_tile(a.s, tile, kChunk, lane);
    if (t.s < 0) return;  // the whole workgroup
    const int count = min(kChunk, t.rows.count - t.row0);
    if (count <= 0) return;
    const size_t first = (size_t)t.rows.first + t.row0;
    const int kh = head / (heads / a.k.heads);

    // rows beyond the last: zero keys, decay 1, beta 0
    const int row = 16 * wave + m;
    h8 kf[NK], qf[NK];
#pragma unroll
    for (int s = 0; s < NK; ++s) {
        kf[s] = qf[s] = (h8){};
        if (row < count) {
            kf[s] = load_h8((const _Float16 *)a.k.data + (first + row) * a.k.token_stride + kh * a.k.head_stride +
                                32 * s + 8 * q, a.k.vec);
            qf[s] = load_h8((const _Float16 *)a.q.data + (first + row) * a.q.token_stride + kh * a.q.head_stride +
                                32 * s + 8 * q, a.q.vec);
        }
    }
    Gates gt{0.f, 0.f};
    if (lane < count) gt = gates_of(a, first + lane, head);
    double G = gt.g;  // 64 bits: differences of long sums are the exponents
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(G, d);
        G += lane >= d ? o : 0.0;
    }
    float kk = 0.f, qq = 0.f, k1 = 0.f;
#pragma unroll
    for (int s = 0; s < NK; ++s) {
        kf_lds[(wave * NK + s) * 64 + lane] = kf[s];
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
        rk = inverse_length(kk, a.eps);
        rq = inverse_length(qq, a.eps);
    }
    if (row >= count) rk = rq = 0.f;  // 1 / sqrt(0) where eps is 0
    if (wave == 0) sum_lds[lane] = G;
    if (q == 0) {
        kr_lds[row] = rk;
        qr_lds[row] = rq * a.scale;
    }
    __syncthreads();

    char *const block = chunks + ((size_t)tile * heads + head) * kChunkBytes;
    f4 kk_acc[4], qk_acc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        kk_acc[j] = qk_acc[j] = (f4){0.f, 0.f, 0.f, 0.f};
        if (j <= wave) {
#pragma unroll
            for (int s = 0; s < NK; ++s) {
                const h8 b = kf_lds[(j * NK + s) * 64 + lane];
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
        const double Gc = sum_lds[c];
        const float kc = kr_lds[c];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = 16 * wave + 4 * q + r;
            float av = 0.f, pv = 0.f;
            if (i >= c) {
                const float fall = decay_of((float)(Gr[r] - Gc)) * kc;
                pv = qr[r] * fall * qk_acc[j][r];
                if (i > c) av = brk[r] * fall * kk_acc[j][r];
            }
            A[i * kRowFloats + c] = av;
            Pm[i * kRowFloats + c] = pv;
            p_most = fmaxf(p_most, __builtin_fabsf(pv));
        }
    }
    p_most = wave_max(p_most);
    if (lane == 0) most_lds[wave] = p_most;
    // row factors and scalars, by the wave that has the rows' k1: each wave its 16, wave 0 all
    const float beta_row = __shfl(gt.beta, row);
    const float since = decay_of((float)__shfl(G, row)) * rk;
    const float l1 = wave_max(__builtin_fabsf(beta_row * since) * k1);
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
    t_most = wave_max(t_most);
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
            const float *const from = (which ? Pm : T) + row_of(wave, m) * kRowFloats + 32 * s + 8 * q;
            const float to = which ? pf.to : tf.to;
            h8 hi, lo;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                _Float16 x, y;
                split(from[j] * to, x, y);
                hi[j] = x;
                lo[j] = y;
                if (!which) t_sum += __builtin_fabsf(from[j]);
            }
            h8 *const at = (h8 *)(block + ((which * kFrags + frag_of(wave, s)) * 2) * kFrag) + lane;
            at[0] = hi;
            at[64] = lo;
        }
    }
    t_sum = wave_max(sum_quarters(t_sum));
    if (lane == 0) sum_T_lds[wave] = t_sum;
    __syncthreads();
    if (wave == 0) {  // lane = row
        const float r = kr_lds[lane], e = decay_of((float)G);
        const float until = decay_of((float)(G_end - G)) * r;
        float *const f = (float *)(block + kRowFactors);
        f[lane] = e * r;
        f[kChunk + lane] = e * qr_lds[lane];
        f[2 * kChunk + lane] = gt.beta;
        f[3 * kChunk + lane] = until;
        const float until_most = wave_max(__builtin_fabsf(until)), beta_most = wave_max(__builtin_fabsf(gt.beta));
        if (lane == 0) {
            const int e_w = __builtin_amdgcn_frexp_expf(until_most);
            const int k = e_w < -110 ? -110 : e_w;
            float *const s = (float *)(block + kScalars);
            s[kDecay] = decay_of((float)G_end);
            // |U| <= (largest row sum of T) |R|: another power of two keeps U where R was
            const int e_u = __builtin_amdgcn_frexp_expf(
                fmaxf(fmaxf(sum_T_lds[0], sum_T_lds[1]), fmaxf(sum_T_lds[2], sum_T_lds[3])));
            s[kUFit] = __builtin_amdgcn_ldexpf(tf.back, -e_u);
            s[kUBack] = __builtin_amdgcn_ldexpf(1.f, e_u);
            s[kPBack] = pf.back;
            s[kWFit] = __builtin_amdgcn_ldexpf(1.f, -k);
            s[kWBack] = __builtin_amdgcn_ldexpf(1.f, k);
            s[kRState] = fmaxf(fmaxf(l1_lds[0], l1_lds[1]), fmaxf(l1_lds[2], l1_lds[3]));
            s[kRValue] = beta_most;
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

// A workgroup of KD / 32 waves has columns 16 slice .. of one head's state; wave w its rows 32 w .. 32 w + 31, as
// two tiles, and TT of the chunk's four row tiles.
template <int KD>
__global__ __launch_bounds__(2 * KD) void delta_scan_kernel(DeltaArgs a, const char *chunks, size_t tiles, int units,
                                                            int slices) {
    constexpr int NW = KD / 32, TT = 4 / NW;
    __shared__ h8 s_lds[NW][2][64];          // the state's operand: 32 rows, high and low
    __shared__ h8 r_lds[2][2][64];           // R's, 32 rows each
    __shared__ h8 u_lds[2][2][64], w_lds[2][2][64];
    __shared__ __attribute__((aligned(16))) _Float16 k_lds[NW][kChunk][32];  // 32 elements of each key
    __shared__ float back_lds[NW][16], v_lds[NW][16];

    // the slices of a head on one XCD, whose L2 then holds what they share
    const int id = blockIdx.x, at_xcd = id >> 3;
    const int unit = at_xcd / slices * 8 + (id & 7), slice = at_xcd % slices;
    if (unit >= units) return;
    const int heads = a.v.heads, s = unit / heads, head = unit - s * heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, q = lane >> 4;
    const int kh = head / (heads / a.k.heads);
    const Rows rows = rows_of(a.s, s);
    const int in = slot_in(a.s, s), out = slot_out(a.s, s);
    const size_t state_size = (size_t)heads * KD * a.value_dim;
    const size_t state_at = ((size_t)head * KD + 32 * wave + 8 * q) * a.value_dim + 16 * slice + m;

    float S[2][4];
    const float start = in == kBadState ? __builtin_nanf("") : 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            S[t][i] = in >= 0 ? a.states[in * state_size + state_at + (size_t)(4 * t + i) * a.value_dim] : start;

    const size_t tile0 = tiles_before(a.s, s, lane);
    // starts that overlap have more chunks than the workspace holds: those are left out
    const int n_chunks = (int)min((size_t)(rows.count + kChunk - 1) / kChunk, tiles - min(tiles, tile0));
    const char *const block0 = chunks + (tile0 * heads + head) * kChunkBytes;
    const size_t step = (size_t)heads * kChunkBytes;

    h8 kf[TT][NW], qf[TT][NW], tf[TT][2][2], pf[TT][2][2];
    f4 fk[TT], fq[TT], fb[TT], fu[TT];
    float v[TT][4];
    auto load_kq = [&](int c) {
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            // a row beyond the last is the last: its factors are 0
            const size_t row = (size_t)rows.first + min(c * kChunk + row_of(wave * TT + tt, m), rows.count - 1);
            const _Float16 *const kp = (const _Float16 *)a.k.data + row * a.k.token_stride + kh * a.k.head_stride + 8 * q;
            const _Float16 *const qp = (const _Float16 *)a.q.data + row * a.q.token_stride + kh * a.q.head_stride + 8 * q;
#pragma unroll
            for (int g = 0; g < NW; ++g) {
                kf[tt][g] = load_h8(kp + 32 * g, a.k.vec);
                qf[tt][g] = load_h8(qp + 32 * g, a.q.vec);
            }
        }
    };
    auto load_v = [&](int c) {
        const float *const f = (const float *)(block0 + c * step + kRowFactors);
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const int r0 = row_of(wave * TT + tt, 4 * q);
            fk[tt] = *(const f4 *)(f + r0);
            fb[tt] = *(const f4 *)(f + 2 * kChunk + r0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const size_t row = (size_t)rows.first + min(c * kChunk + r0 + i, rows.count - 1);
                v[tt][i] = (float)((const _Float16 *)a.v.data)[row * a.v.token_stride + head * a.v.head_stride + 16 * slice + m];
            }
        }
    };
    auto load_matrix = [&](int c, int which, h8 (&to)[TT][2][2]) {
        const h8 *const p = (const h8 *)(block0 + c * step + which * kFrags * 2 * kFrag) + lane;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const int t = wave * TT + tt;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                if (g > t >> 1) continue;
                to[tt][g][0] = p[frag_of(t, g) * 128];
                to[tt][g][1] = p[frag_of(t, g) * 128 + 64];
            }
        }
    };
    auto load_u = [&](int c, int which, f4 (&to)[TT]) {
        const float *const f = (const float *)(block0 + c * step + kRowFactors) + which * kChunk;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) to[tt] = *(const f4 *)(f + row_of(wave * TT + tt, 4 * q));
    };
    if (n_chunks) {
        load_kq(0);
        load_v(0);
        load_matrix(0, 0, tf);
        load_u(0, 3, fu);
        load_matrix(0, 1, pf);
        load_u(0, 1, fq);
    }
    const f4 zero = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < n_chunks; ++c) {
        const int next = min(c + 1, n_chunks - 1);
        const float *const scalar = (const float *)(block0 + c * step + kScalars);
        const float decay = scalar[kDecay], u_fit = scalar[kUFit], u_more = scalar[kUBack], p_back = scalar[kPBack];
        const float w_fit = scalar[kWFit], w_back = scalar[kWBack], r_state = scalar[kRState], r_value = scalar[kRValue];

        // the state as an operand, each wave's rows by their own power of two a column
        float top = 0.f, v_top = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, __builtin_fabsf(S[t][i]));
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) v_top = fmaxf(v_top, __builtin_fabsf(v[tt][i]));
        top = max_quarters(top);
        v_top = max_quarters(v_top);
        const Fit sf = fit_of(top);
        h8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            _Float16 x, y;
            split(S[j / 4][j % 4] * sf.to, x, y);
            hi[j] = x;
            lo[j] = y;
        }
        s_lds[wave][0][lane] = hi;
        s_lds[wave][1][lane] = lo;
        if (q == 0) {
            back_lds[wave][m] = sf.back;
            v_lds[wave][m] = v_top;
        }
        lds_barrier();

        // K S and Q S; the keys go to LDS for the update
        f4 ks[TT], qs[TT];
        float s_back = 0.f, v_most = 0.f;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) ks[tt] = qs[tt] = zero;
#pragma unroll
        for (int g = 0; g < NW; ++g) {
            const h8 b_hi = s_lds[g][0][lane], b_lo = s_lds[g][1][lane];
            const float back = back_lds[g][m];
            s_back = fmaxf(s_back, back);
            v_most = fmaxf(v_most, v_lds[g][m]);
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                const f4 x = mfma16(kf[tt][g], b_lo, mfma16(kf[tt][g], b_hi, zero));
                const f4 y = mfma16(qf[tt][g], b_lo, mfma16(qf[tt][g], b_hi, zero));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    ks[tt][i] = __builtin_fmaf(x[i], back, ks[tt][i]);
                    qs[tt][i] = __builtin_fmaf(y[i], back, qs[tt][i]);
                }
            }
        }
#pragma unroll
        for (int tt = 0; tt < TT; ++tt)
#pragma unroll
            for (int g = 0; g < NW; ++g)
                *(h8 *)&k_lds[g][row_of(wave * TT + tt, m)][8 * (q ^ (m >> 2))] = kf[tt][g];
        load_kq(next);

        // R = beta (V - e^G K S), |R| <= r_value |V| + r_state |S|
        const Fit rf = fit_of(__builtin_fmaf(r_value, v_most, r_state * (s_back * 32768.f)));
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            h4 r_hi, r_lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float r = fb[tt][i] * (v[tt][i] - fk[tt][i] * ks[tt][i]);
                _Float16 x, y;
                split(r * rf.to, x, y);
                r_hi[i] = x;
                r_lo[i] = y;
            }
            const int t = wave * TT + tt;
            *((h4 *)&r_lds[t >> 1][0][lane] + (t & 1)) = r_hi;
            *((h4 *)&r_lds[t >> 1][1][lane] + (t & 1)) = r_lo;
        }
        load_v(next);
        lds_barrier();

        // U = T R
        const float u_back = rf.back * u_more;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const int t = wave * TT + tt;
            f4 x = zero, y = zero;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                if (g > t >> 1) continue;
                const h8 b_hi = r_lds[g][0][lane], b_lo = r_lds[g][1][lane];
                x = mfma16(tf[tt][g][0], b_hi, x);
                y = mfma16(tf[tt][g][0], b_lo, y);
                y = mfma16(tf[tt][g][1], b_hi, y);
            }
            h4 u_hi, u_lo, w_hi, w_lo;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = (x[i] + y[i]) * u_fit;
                _Float16 e, f;
                split(u * (fu[tt][i] * w_fit), e, f);
                w_hi[i] = e;
                w_lo[i] = f;
                split(u, e, f);
                u_hi[i] = e;
                u_lo[i] = f;
            }
            *((h4 *)&w_lds[t >> 1][0][lane] + (t & 1)) = w_hi;
            *((h4 *)&w_lds[t >> 1][1][lane] + (t & 1)) = w_lo;
            *((h4 *)&u_lds[t >> 1][0][lane] + (t & 1)) = u_hi;
            *((h4 *)&u_lds[t >> 1][1][lane] + (t & 1)) = u_lo;
        }
        load_matrix(next, 0, tf);
        load_u(next, 3, fu);
        lds_barrier();

        // S <- e^G_64 S + K^T W
        f4 acc[2] = {zero, zero};
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const h8 b_hi = w_lds[g][0][lane], b_lo = w_lds[g][1][lane];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                // 16 lanes read four keys' elements 8 c + 4 t .. + 3 (c < 4): lane m gets column m of them
                const _Float16 *const at = &k_lds[wave][32 * g + 8 * q + (m >> 2)][8 * ((m & 3) ^ q) + 4 * t];
                const h4 k0 = bitcast<h4>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)at));
                const h4 k1 = bitcast<h4>(__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(at + 4 * 32)));
                const h8 kt = {k0[0], k0[1], k0[2], k0[3], k1[0], k1[1], k1[2], k1[3]};
                acc[t] = mfma16(kt, b_lo, mfma16(kt, b_hi, acc[t]));
            }
        }
        const float back = u_back * w_back;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) S[t][i] = __builtin_fmaf(acc[t][i], back, decay * S[t][i]);

        // out = e^G Q S + P U
        const float o_back = u_back * p_back;
#pragma unroll
        for (int tt = 0; tt < TT; ++tt) {
            const int t = wave * TT + tt;
            f4 x = zero, y = zero;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                if (g > t >> 1) continue;
                const h8 b_hi = u_lds[g][0][lane], b_lo = u_lds[g][1][lane];
                x = mfma16(pf[tt][g][0], b_hi, x);
                y = mfma16(pf[tt][g][0], b_lo, y);
                y = mfma16(pf[tt][g][1], b_hi, y);
            }
            const int r0 = c * kChunk + row_of(t, 4 * q);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float o = __builtin_fmaf(x[i] + y[i], o_back, fq[tt][i] * qs[tt][i]);
                if (r0 + i < rows.count)
                    ((_Float16 *)a.out.data)[((size_t)rows.first + r0 + i) * a.out.token_stride +
                                             head * a.out.head_stride + 16 * slice + m] = (_Float16)o;
            }
        }
        load_matrix(next, 1, pf);
        load_u(next, 1, fq);
    }
    if (out >= 0) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                a.states[out * state_size + state_at + (size_t)(4 * t + i) * a.value_dim] = S[t][i];
    }
}

template <int KD>
hipError_t launch_kd(const DeltaArgs &a, char *chunks, hipStream_t stream) {
    const size_t tiles = tile_count(a.s, kChunk);
    delta_prepare_kernel<KD><<<dim3((unsigned)(tiles * a.v.heads)), dim3(256), 0, stream>>>(a, chunks);
    const int units = a.s.sequences * a.v.heads, slices = a.value_dim / 16;
    const unsigned blocks = (unsigned)((units + 7) / 8 * 8 * slices);
    delta_scan_kernel<KD><<<dim3(blocks), dim3(2 * KD), 0, stream>>>(a, chunks, tiles, units, slices);
    return hipGetLastError();
}

}  // namespace

size_t delta_prompt_bytes(size_t heads, size_t sequences, size_t tokens) {
    if (tokens < kDeltaPromptRows * sequences) return 0;
    return kSharedPrefixBytes + (tokens / kChunk + sequences) * heads * kChunkBytes;
}

hipError_t launch_delta_prompt(const DeltaArgs &a, void *workspace, hipStream_t stream) {
    char *const chunks = (char *)workspace + kSharedPrefixBytes;
    return a.key_dim == 64 ? launch_kd<64>(a, chunks, stream) : launch_kd<128>(a, chunks, stream);
}

}  // namespace exl3k

// exl3_attention_cached.hip -- attention of each sequence's last tokens over the quantised cache.
#include "exl3_attention_rows.hpp"
#include "exl3_launch.hpp"

namespace exl3k {

namespace {

template <int D, int BITS>
struct CachedRows {
    const uint8_t *pages;
    const int32_t *table;
    size_t page_count;
    KvLayout l;
    int head;
    __device__ const uint8_t *at(int n) const {
        const int page = table[n / l.page_tokens];
        if (page < 0 || (size_t)page >= page_count) return nullptr;
        return pages + (size_t)page * l.page_bytes + (size_t)head * l.region;
    }
    __device__ static float code(uint8_t b, int i) {
        return BITS == 8 ? (float)((int)b - 128) : (float)((int)((i & 1) ? b >> 4 : b & 15) - 8);
    }
    __device__ float key(int n, int i) const {
        const uint8_t *b = at(n);
        if (!b) return __builtin_nanf("");
        const int t = n % l.page_tokens;
        const float s = half_bits_to_float(((const uint16_t *)(b + l.ks_off))[t * (D / 32) + i / 32]);
        return code(b[(size_t)t * (D * BITS / 8) + i * BITS / 8], i) * s;
    }
    __device__ float value(int n, int i) const {
        const uint8_t *b = at(n);
        if (!b) return __builtin_nanf("");
        const int t = n % l.page_tokens;
        const float s = half_bits_to_float(((const uint16_t *)(b + l.vs_off))[(t / 4 * (D / 32) + i / 32) * 4 + t % 4]);
        constexpr int PART = D * BITS / 128, W = D / 16;
        return code(b[l.v_off + (size_t)(t / 4) * (D * BITS / 2) + i / W * (4 * PART) + t % 4 * PART + i % W * BITS / 8], i) * s;
    }
};

// One wave per query row and head.
template <int D, int BITS>
__global__ __launch_bounds__(64) void attention_cached_kernel(CachedArgs a) {
    const int row = blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
    const int s = row / a.q_len, j = row - s * a.q_len;
    const long most = (long)a.table_stride * a.l.page_tokens;
    long n = a.kv_lens[s];
    n = n > most ? most : n;
    const int seen = (int)n - (a.q_len - 1 - j);
    const CachedRows<D, BITS> r{a.pages, a.page_table + (size_t)s * a.table_stride, a.page_count, a.l,
                                head / (a.q.heads / a.l.kv_heads)};
    float o[D / 64];
    const float inv = attend_row<D>((const _Float16 *)a.q.data + (size_t)row * a.q.token_stride + head * a.q.head_stride,
                                    1, r, seen, a.scale, o);
    __shared__ float os[D];
    for (int i = 0; i < D / 64; ++i) os[i * 64 + lane] = o[i] * inv;
    __syncthreads();
    if (8 * lane < D) {
        float x[8];
        for (int e = 0; e < 8; ++e) x[e] = os[8 * lane + e];
        h32_run8(x, lane);
        store_run8<1>(a.out.data, (size_t)row * a.out.token_stride + head * a.out.head_stride + 8 * lane, a.out.vec, x);
    }
}

}  // namespace

size_t attention_cached_bytes(size_t q_heads, size_t kv_heads, size_t head_dim, size_t sequences, size_t q_len) {
    (void)q_heads, (void)kv_heads, (void)head_dim, (void)sequences, (void)q_len;
    return kSharedPrefixBytes;
}

hipError_t launch_attention_cached(const CachedArgs &a, void *workspace, hipStream_t stream) {
    (void)workspace;
    const dim3 grid(a.sequences * a.q_len, a.q.heads);
    const int bits = a.l.bits;
    if (a.l.head_dim == 64) {
        if (bits == 4) attention_cached_kernel<64, 4><<<grid, 64, 0, stream>>>(a);
        else attention_cached_kernel<64, 8><<<grid, 64, 0, stream>>>(a);
    } else if (a.l.head_dim == 128) {
        if (bits == 4) attention_cached_kernel<128, 4><<<grid, 64, 0, stream>>>(a);
        else attention_cached_kernel<128, 8><<<grid, 64, 0, stream>>>(a);
    } else {
        if (bits == 4) attention_cached_kernel<256, 4><<<grid, 64, 0, stream>>>(a);
        else attention_cached_kernel<256, 8><<<grid, 64, 0, stream>>>(a);
    }
    return hipGetLastError();
}

}  // namespace exl3k

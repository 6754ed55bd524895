// Attention of a batch's tokens over a paged cache.
#include "device_util.h"
#include "paged.h"

namespace th {

namespace {

__device__ __forceinline__ float load_kv(const float *p) { return *p; }
__device__ __forceinline__ float load_kv(const uint16_t *p) { return bf16_to_f32(*p); }

// One wave a (token, head), a key at a time.
template <int HD, typename KV>
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedAttnArgs a) {
    constexpr int E = HD / 64;
    const int lane = threadIdx.x & 63;
    const size_t item = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const size_t t = item / a.n_heads;
    if (t >= a.b.head->n_tokens) return;
    const int h = (int)(item % a.n_heads), g = h / a.group;
    const TokenAt at = a.b.tokens[t];
    const SeqAt seq = a.b.seqs[at.seq];
    float q[E], acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = a.q[item * HD + lane + 64 * e];
        acc[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const uint32_t mask = (1u << a.b.page_shift) - 1;
    for (uint32_t j = 0; j <= seq.context + at.index; ++j) {
        if (j >= seq.context && seq.is_tree) {
            const uint32_t d = j - seq.context;
            if (!(a.b.tree[t * kTreeWords + d / 64] >> (d & 63) & 1)) continue;
        }
        const size_t page = a.b.pages[seq.page0 + (j >> a.b.page_shift)];
        const KV *k = static_cast<const KV *>(a.cache) + (((page * 2 * a.n_kv_heads + g) << a.b.page_shift) + (j & mask)) * HD;
        const KV *v = k + ((size_t)a.n_kv_heads << a.b.page_shift) * HD;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(q[e], load_kv(k + lane + 64 * e), s);
        s = wave_sum(s) * a.scale;
        const float m_new = fmaxf(m, s);
        const float alpha = m == -INFINITY ? 0.f : expf(m - m_new), p = s == -INFINITY ? 0.f : expf(s - m_new);
        l = l * alpha + p;
        m = m_new;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(p, load_kv(v + lane + 64 * e), acc[e] * alpha);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) a.out[item * HD + lane + 64 * e] = acc[e] / l;
}

template <int HD>
hipError_t attention(hipStream_t s, const PagedAttnArgs &a, size_t n, bool bf16) {
    const unsigned grid = (unsigned)((n * a.n_heads + 3) / 4);
    if (bf16) paged_attention_kernel<HD, uint16_t><<<grid, 256, 0, s>>>(a);
    else paged_attention_kernel<HD, float><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_attention(hipStream_t s, const PagedAttnArgs &a, size_t n, size_t head_dim, bool bf16) {
    if (n == 0) return hipSuccess;
    return head_dim == 64    ? attention<64>(s, a, n, bf16)
           : head_dim == 128 ? attention<128>(s, a, n, bf16)
                             : attention<256>(s, a, n, bf16);
}

}  // namespace th

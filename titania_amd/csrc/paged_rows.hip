// Kernels over the rows of paged caches and batches: the append (head norms,
// rotation and cache write in one pass), the rows of accepted tokens moved up,
// the argmax of many rows, and a batch's arrays from pinned memory.
#include "device_util.h"
#include "paged.h"
#include "q8.h"

namespace th {

namespace {

__device__ __forceinline__ void store_kv4(float *p, const float4 &v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void store_kv4(uint16_t *p, const float4 &v) {
    *reinterpret_cast<uint2 *>(p) =
        make_uint2(f32_to_bf16(v.x) | (uint32_t)f32_to_bf16(v.y) << 16, f32_to_bf16(v.z) | (uint32_t)f32_to_bf16(v.w) << 16);
}

// The sum over aligned groups of `LANES` lanes, in each of them.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Of a head's values x: x / sqrt(mean(x^2) + eps) times the gains, then of each
// pair (a, b) = (x_i, x_{i + HD/2}): (a cos - b sin, b cos + a sin). HD / 8 lanes
// a head: a lane has four neighbouring values of each half, so that a rotation's
// pairs are its own. Bound by HBM: 7129 tokens of 32 / 8 heads to a bf16 cache
// 61 us, 5.3 TB/s; one token 2.5 us, a launch.
template <int HD, typename KV>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
    constexpr int LPH = HD / 8, HPB = 256 / LPH;
    const int sub = threadIdx.x % LPH;
    const uint32_t unit = blockIdx.x * HPB + threadIdx.x / LPH;
    const uint32_t heads = a.n_heads + 2 * a.n_kv_heads;
    const uint32_t t = unit / heads;
    if (t >= a.b.head->n_tokens) return;
    int h = (int)(unit % heads);
    const TokenAt at = a.b.tokens[t];
    const bool is_q = h < a.n_heads, is_v = h >= a.n_heads + a.n_kv_heads;
    if (!is_q) h -= a.n_heads + (is_v ? a.n_kv_heads : 0);
    const float *src = (is_q ? a.q : is_v ? a.v : a.k) + ((size_t)t * (is_q ? a.n_heads : a.n_kv_heads) + h) * HD;
    float4 x = reinterpret_cast<const float4 *>(src)[sub], y = reinterpret_cast<const float4 *>(src + HD / 2)[sub];
    if (!is_v) {
        const uint16_t *gain = is_q ? a.q_norm : a.k_norm;
        if (gain) {
            float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w + y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w;
            ss = lanes_sum<LPH>(ss);
            const float r = 1.0f / sqrtf(ss / HD + a.eps);
            const uint2 g = reinterpret_cast<const uint2 *>(gain)[sub], f = reinterpret_cast<const uint2 *>(gain + HD / 2)[sub];
            x = make_float4(x.x * r * bf16_lo(g.x), x.y * r * bf16_hi(g.x), x.z * r * bf16_lo(g.y), x.w * r * bf16_hi(g.y));
            y = make_float4(y.x * r * bf16_lo(f.x), y.y * r * bf16_hi(f.x), y.z * r * bf16_lo(f.y), y.w * r * bf16_hi(f.y));
        }
        const float4 *cs = reinterpret_cast<const float4 *>(a.rope + (size_t)at.pos * HD) + 2 * sub;
        const float4 c = cs[0], d = cs[1];  // (cos, sin) of two pairs each
        const float4 u = x, w = y;
        x = make_float4(u.x * c.x - w.x * c.y, u.y * c.z - w.y * c.w, u.z * d.x - w.z * d.y, u.w * d.z - w.w * d.w);
        y = make_float4(w.x * c.x + u.x * c.y, w.y * c.z + u.y * c.w, w.z * d.x + u.z * d.y, w.w * d.z + u.w * d.w);
    }
    if (is_q) {
        float *dst = a.q_out + ((size_t)t * a.n_heads + h) * HD;
        reinterpret_cast<float4 *>(dst)[sub] = x;
        reinterpret_cast<float4 *>(dst + HD / 2)[sub] = y;
        return;
    }
    const uint32_t page = at.slot >> a.b.page_shift, row = at.slot & ((1u << a.b.page_shift) - 1);
    KV *dst = reinterpret_cast<KV *>(a.cache) +
              (((((size_t)page * 2 + is_v) * a.n_kv_heads + h) << a.b.page_shift) + row) * HD;
    store_kv4(dst + 4 * sub, x);
    store_kv4(dst + HD / 2 + 4 * sub, y);
}

template <int HD>
hipError_t append(hipStream_t s, const PagedAppendArgs &a, size_t n, bool bf16) {
    constexpr size_t kHeads = 256 / (HD / 8);
    const unsigned grid = (unsigned)((n * (a.n_heads + 2 * a.n_kv_heads) + kHeads - 1) / kHeads);
    if (bf16) paged_append_kernel<HD, uint16_t><<<grid, 256, 0, s>>>(a);
    else paged_append_kernel<HD, float><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

// A thread takes 16 bytes of each moved row, of one head's keys or values, so
// that no other thread reads or writes them. A sequence's moves go up to row j
// from row i_j >= j, the i_j rising: what move j reads is no target of an
// earlier one, and may be that of a later one. Reading eight rows before
// writing them keeps that order. The moves are the launch's arguments, so that
// nothing is copied before it: a tree in 28 layers 3.4 us, a launch.
__global__ __launch_bounds__(256) void paged_moves_kernel(PagedMoves m) {
    const uint32_t per_row = (uint32_t)m.row_bytes / 16;
    const uint32_t unit = blockIdx.x * 256 + threadIdx.x;
    const uint32_t kv_head = unit / per_row;  // of the keys', then the values'
    if (kv_head >= 2u * m.n_kv_heads) return;
    const uint32_t mask = (1u << m.page_shift) - 1;
    th_u32x4 *const base = static_cast<th_u32x4 *>(m.cache[blockIdx.z]) + unit % per_row;
    const int shift = m.page_shift, halves = 2 * m.n_kv_heads;
    auto at = [=](uint32_t slot) {
        const size_t r = (((size_t)(slot >> shift) * halves + kv_head) << shift) + (slot & mask);
        return base + r * per_row;
    };
    const uint32_t end = m.start[blockIdx.y + 1];
    for (uint32_t i = m.start[blockIdx.y]; i < end; i += 8) {
        th_u32x4 v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = *at(m.move[min(i + k, end - 1)].from);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i + k < end) *at(m.move[i + k].to) = v[k];
    }
}

// One block a part of a row, 16 bytes a lane and load, eight in flight. Bound by
// HBM: 462 rows of 151936 57 us, 4.9 TB/s, 24 rows 6.4.
__global__ __launch_bounds__(256) void argmax_rows_kernel(const float *x, size_t cols, int splits, size_t part,
                                                          uint64_t *picks) {
    __shared__ uint64_t red[4];
    const size_t row = blockIdx.x / splits, split = blockIdx.x % splits;
    const size_t c0 = split * part, c1 = c0 + part < cols ? c0 + part : cols;
    const float *r = x + row * cols;
    uint64_t best = 0;
    for (size_t c = c0 + 4 * threadIdx.x; c < c1; c += 8 * 1024) {
        f32x4_any v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c + 1024 * k + 4 <= c1) v[k] = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any *>(r + c + 1024 * k));
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const size_t at = c + 1024 * k;
            if (at + 4 <= c1) {
#pragma unroll
                for (int e = 0; e < 4; ++e) best = max_u64(best, argmax_pack(v[k][e], (uint32_t)(at + e)));
            } else {
                for (size_t e = at; e < c1; ++e) best = max_u64(best, argmax_pack(r[e], (uint32_t)e));
            }
        }
    }
    best = wave_max_u64(best);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = best;
    __syncthreads();
    if (threadIdx.x == 0) picks[blockIdx.x] = max_u64(max_u64(red[0], red[1]), max_u64(red[2], red[3]));
}

__global__ __launch_bounds__(256) void upload_kernel(Upload u) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
        for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < u.units[k]; i += gridDim.x * 256)
            static_cast<uint4 *>(u.to[k])[i] = static_cast<const uint4 *>(u.from[k])[i];
}

}  // namespace

hipError_t launch_paged_append(hipStream_t s, const PagedAppendArgs &a, size_t n, size_t head_dim, bool bf16) {
    if (n == 0) return hipSuccess;
    return head_dim == 64 ? append<64>(s, a, n, bf16) : head_dim == 128 ? append<128>(s, a, n, bf16) : append<256>(s, a, n, bf16);
}

hipError_t launch_paged_moves(hipStream_t s, const PagedMoves &m) {
    const unsigned units = 2u * m.n_kv_heads * (m.row_bytes / 16);
    paged_moves_kernel<<<dim3((units + 255) / 256, m.n_segments, m.n_layers), 256, 0, s>>>(m);
    return hipGetLastError();
}

hipError_t launch_argmax_rows(hipStream_t s, const float *x, size_t rows, size_t cols, const RowParts &parts, uint64_t *picks) {
    argmax_rows_kernel<<<(unsigned)(rows * parts.splits), 256, 0, s>>>(x, cols, (int)parts.splits, parts.part, picks);
    return hipGetLastError();
}

hipError_t launch_upload(hipStream_t s, const Upload &u) {
    uint32_t most = 0;
    for (uint32_t n : u.units) most = std::max(most, n);
    upload_kernel<<<std::min(64u, (most + 255) / 256 + 1), 256, 0, s>>>(u);
    return hipGetLastError();
}

}  // namespace th

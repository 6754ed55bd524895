// Attention of a batch's tokens over a paged cache, as the batch's plan cuts
// it: tiles of rows (a token and a query head of the KV head's group), over all
// positions that they see or a part of them. Partial results are joined by a
// second launch.
#include <algorithm>
#include <type_traits>

#include "device_util.h"
#include "paged.h"

namespace th {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kFewThreads = 256;

// 16 bytes of a cached row as f32.
__device__ __forceinline__ void widen(const th_u32x4 &w, float (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void widen(const th_u32x4 &w, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = bf16_lo(w[i]);
        f[2 * i + 1] = bf16_hi(w[i]);
    }
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void widen(const u32x2 &w, float (&f)[4]) {  // four of 16 bits
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        f[2 * i] = bf16_lo(w[i]);
        f[2 * i + 1] = bf16_hi(w[i]);
    }
}

__device__ __forceinline__ bool finite(float f) { return (__float_as_uint(f) & 0x7f800000u) != 0x7f800000u; }

// Which of the 16 positions from c on a sequence's token sees, a bit each.
// Selects, no branches of single lanes.
__device__ __forceinline__ uint32_t seen16(const SeqAt &seq, const uint64_t *tree, uint32_t token, uint32_t c) {
    const int d = (int)(c - seq.context);  // of the first; negative: in the context
    const int before = d < 0 ? -d : 0;     // (at most 15 where this is called)
    if (!seq.is_tree) {
        const int n = (int)token + 1 - d;
        return n <= 0 ? 0u : n >= 16 ? 0xffffu : (1u << n) - 1;
    }
    const uint64_t *words = tree + (size_t)(seq.token0 + token) * kTreeWords;
    const int at = d < 0 ? 0 : d, word = at >> 6, shift = at & 63;
    const uint64_t low = words[word] >> shift, high = words[word + 1 < kTreeWords ? word + 1 : word];
    const uint32_t bits = (uint32_t)low | (shift > 48 && word + 1 < kTreeWords ? (uint32_t)(high << (64 - shift)) : 0u);
    return ((bits << before) | ((1u << before) - 1)) & 0xffffu;
}

// Tiles of up to 16 R rows. Each of four waves takes 16 of every 64 positions
// on its own, with no barrier before the end: keys and values go from memory
// straight into the operands of v_mfma_f32_16x16x4_f32, whose products and
// sums are those of f32, so nothing is converted or lost and any value counts
// as it is.
//
// S^T = K Q^T (16 positions down, 16 rows across): lane (m, g) = (lane % 16,
// lane / 16) has key m's values of every fourth 16 bytes, g of each 64 (the
// order in which a sum's products are formed is free, so that loads are whole
// 16 bytes), and Q's in the same order. The result leaves the lane positions
// 4 g + {0..3} of row m: masks, maximum and exponentials are the lane's own but
// for two exchanges, and the weights are, register by register, the operand of
// O^T = V^T P^T with positions 4 g + i at step i, for which the lane loads
// those rows of V.
//
// A step's 64 products of 32 cycles take a wave 2048 cycles a row set, while
// the block's 64 KB of f32 keys and values take a CU's share of HBM 8000: up to
// 64 rows cost what one costs (32 with a bf16 cache).
template <int HD, int R, typename KV>
__global__ __launch_bounds__(kFewThreads, R == 1 && HD < 256 ? 2 : 1) void paged_few_kernel(PagedAttnArgs a, int cls) {
    constexpr int VE = 16 / sizeof(KV);         // values of 16 bytes
    constexpr int KJ = HD / (4 * VE);           // 16-byte loads of a lane's part of a key
    constexpr int VV = VE <= HD / 16 ? VE : HD / 16;  // values of a load of a value row, which 16 lanes share
    constexpr int VJ = HD / (16 * VV);          // such loads
    using VLoad = std::conditional_t<VV == VE, th_u32x4, u32x2>;
    constexpr int QS = HD + 4;                  // floats between rows of Q in LDS
    constexpr int kMerge = 4 * 16 * (HD + 4);   // the waves' results of 16 rows
    constexpr int kLds = R * 16 * QS > kMerge ? R * 16 * QS : kMerge;
    __shared__ __align__(16) float lds[kLds];
    __shared__ float stat[4][16 * R][2];
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t first = a.b.head->first[cls], n = (a.b.head->first[cls + 1] - first) * a.n_kv_heads;
    const float c2 = a.scale * kLog2e;
    for (uint32_t at = blockIdx.x; at < n; at += gridDim.x) {
        const ItemAt it = a.b.items[first + at / a.n_kv_heads];
        const int kvh = at % a.n_kv_heads;
        const SeqAt seq = a.b.seqs[it.seq];
        const uint32_t rows = min((uint32_t)(16 * R), seq.n_new * a.group - it.row0);
        const float *const qb = a.q + ((size_t)seq.token0 * a.n_heads + (size_t)kvh * a.group) * HD;
        // Row `row` of the sequence, in q and out.
        auto row_at = [&](uint32_t row) { return ((size_t)(row / a.group) * a.n_heads + row % a.group) * HD; };
        for (int i = threadIdx.x; i < 16 * R * (HD / 4); i += kFewThreads) {
            const uint32_t r = i / (HD / 4), c = i % (HD / 4);  // rows past the last repeat it
            *reinterpret_cast<float4 *>(&lds[r * QS + 4 * c]) =
                *reinterpret_cast<const float4 *>(qb + row_at(it.row0 + min(r, rows - 1)) + 4 * c);
        }
        uint32_t token[R];
#pragma unroll
        for (int r = 0; r < R; ++r) token[r] = (it.row0 + min((uint32_t)(16 * r + m), rows - 1)) / a.group;
        __syncthreads();
        // Q's operands: of one row set in registers, of more from LDS each time.
        float qr[R == 1 ? KJ : 1][VE];
        auto load_q = [&](int r, int j, float (&f)[VE]) {
#pragma unroll
            for (int e = 0; e < VE; e += 4)
                *reinterpret_cast<float4 *>(&f[e]) =
                    *reinterpret_cast<const float4 *>(&lds[(16 * r + m) * QS + j * 4 * VE + g * VE + e]);
        };
        if constexpr (R == 1)
#pragma unroll
            for (int j = 0; j < KJ; ++j) load_q(0, j, qr[j]);
        f32x4 o[R][HD / 16];
        float mx[R], l[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mx[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) o[r][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        const uint32_t *const pages = a.b.pages + seq.page0;
        const uint32_t mask = (1u << a.b.page_shift) - 1;
        // 16 positions from c on, a multiple of 16, lie in one page.
        auto page_of = [&](uint32_t c) { return pages[min(c, it.k1 - 1) >> a.b.page_shift]; };
        auto rows_of = [&](uint32_t page, uint32_t c) {
            return static_cast<const KV *>(a.cache) +
                   ((((size_t)page * 2 * a.n_kv_heads + kvh) << a.b.page_shift) + (c & mask)) * HD;
        };
        const size_t to_v = ((size_t)a.n_kv_heads << a.b.page_shift) * HD;
        th_u32x4 k[KJ];
        VLoad v[4][VJ];
        auto fetch = [&](uint32_t page, uint32_t c) {
            const KV *kr = rows_of(page, c) + m * HD + g * VE;
            const KV *vr = rows_of(page, c) + to_v + 4 * g * HD + m * VV;
#pragma unroll
            for (int j = 0; j < KJ; ++j) k[j] = *reinterpret_cast<const th_u32x4 *>(kr + j * 4 * VE);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < VJ; ++j) v[i][j] = *reinterpret_cast<const VLoad *>(vr + i * HD + j * 16 * VV);
        };
        uint32_t c = it.k0 + 16 * wave, next = 0;
        if (c < it.k1) {
            fetch(page_of(c), c);
            next = page_of(c + 64);
        }
        for (; c < it.k1; c += 64) {
            float kf[KJ][VE], vf[4][VJ][VV];
#pragma unroll
            for (int j = 0; j < KJ; ++j) widen(k[j], kf[j]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < VJ; ++j) widen(v[i][j], vf[i][j]);
            if (c + 64 < it.k1) {
                fetch(next, c + 64);
                next = page_of(c + 128);
            }
            // Where not every row sees every position: behind the context.
            const bool partly = c + 16 > seq.context;
            uint64_t odd = 0;  // lanes with an infinity or a NaN in a value that some row may not see
            if (partly) {
                bool here = false;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = c + 4 * g + i < it.k1;  // rows behind the last position hold anything
#pragma unroll
                    for (int j = 0; j < VJ; ++j)
#pragma unroll
                        for (int e = 0; e < VV; ++e) {
                            const bool f = finite(vf[i][j][e]);
                            here = here || (in && !f);
                            vf[i][j][e] = in && f ? vf[i][j][e] : 0.f;
                        }
                }
                odd = __ballot(here);
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                // One row set's operands and scores at a time.
                if constexpr (R > 1) asm volatile("" ::: "memory");
                f32x4 s{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < KJ; ++j) {
                    float q[VE];
                    if constexpr (R == 1) {
#pragma unroll
                        for (int e = 0; e < VE; ++e) q[e] = qr[j][e];
                    } else {
                        load_q(r, j, q);
                    }
#pragma unroll
                    for (int e = 0; e < VE; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j][e], q[e], s, 0, 0, 0);
                }
                float x[4], top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = s[i] * c2;
                uint32_t seen = 0xffff;
                if (partly) {
                    seen = seen16(seq, a.b.tree, token[r], c) & (it.k1 - c < 16 ? (1u << (it.k1 - c)) - 1 : 0xffffu);
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = seen >> (4 * g + i) & 1 ? x[i] : -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) top = max_nn(top, x[i]);
                top = max_nn(mx[r], rows_max_nn(top));
                const float base = top == -INFINITY ? 0.f : top;
                if (__any(top != mx[r])) {
                    const float alpha = __builtin_amdgcn_exp2f(mx[r] - base);
                    l[r] *= alpha;
#pragma unroll
                    for (int d = 0; d < HD / 16; ++d) o[r][d] *= alpha;
                    mx[r] = top;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[i] = __builtin_amdgcn_exp2f(x[i] - base);
                    l[r] += s[i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int d = 0; d < HD / 16; ++d)
                        o[r][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[i][d / VV][d % VV], s[i], o[r][d], 0, 0, 0);
                // Values that are no numbers, which the products left out: for
                // the rows that see them alone.
                if (__builtin_expect(odd != 0, 0)) {
#pragma unroll 1
                    for (int key = 0; key < 16 && c + key < it.k1; ++key) {
                        if (!(odd >> (key & ~3) * 4 & 0xffff)) continue;
                        const KV *vr = rows_of(page_of(c), c) + to_v + key * HD;
                        const float mine = (key & 2) ? ((key & 1) ? s[3] : s[2]) : ((key & 1) ? s[1] : s[0]);
                        const float p = __shfl(mine, (key >> 2) * 16 + m, 64);
                        if (!(seen >> key & 1)) continue;
#pragma unroll
                        for (int d = 0; d < HD / 16; ++d)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const KV w = vr[(d / VV) * 16 * VV + (4 * g + i) * VV + d % VV];
                                const float f = sizeof(KV) == 4 ? (float)w : bf16_to_f32((uint16_t)w);
                                if (!finite(f)) o[r][d][i] = fmaf(p, f, o[r][d][i]);
                            }
                    }
                }
            }
        }
        // The four waves' results: o[r][d][i] is dimension (d / VV) 16 VV +
        // (4 g + i) VV + d % VV of row m.
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] = rows_sum(l[r]);
            if (g == 0) {
                stat[wave][16 * r + m][0] = mx[r];
                stat[wave][16 * r + m][1] = l[r];
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (16u * r >= rows) break;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w][16 * r + m][0]);
            const float f = mx[r] == -INFINITY ? (l[r] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(mx[r] - top);
#pragma unroll
            for (int d = 0; d < HD / 16; d += 4)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<float4 *>(
                        &lds[(wave * 16 + m) * (HD + 4) + (d / VV) * 16 * VV + (4 * g + i) * VV + d % VV]) =
                        make_float4(o[r][d][i] * f, o[r][d + 1][i] * f, o[r][d + 2][i] * f, o[r][d + 3][i] * f);
            __syncthreads();
            for (int i = threadIdx.x; i < 16 * (HD / 4); i += kFewThreads) {
                const uint32_t row = i / (HD / 4), col = 4 * (i % (HD / 4));
                if (16 * r + row >= rows) break;
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                float ms = -INFINITY, ls = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) ms = fmaxf(ms, stat[w][16 * r + row][0]);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float4 x = *reinterpret_cast<const float4 *>(&lds[(w * 16 + row) * (HD + 4) + col]);
                    sum = make_float4(sum.x + x.x, sum.y + x.y, sum.z + x.z, sum.w + x.w);
                    const float mw = stat[w][16 * r + row][0], lw = stat[w][16 * r + row][1];
                    ls += mw == -INFINITY ? lw : lw * __builtin_amdgcn_exp2f(mw - ms);
                }
                if (it.part == kNoPart) {
                    float *dst = a.out + ((size_t)seq.token0 * a.n_heads + (size_t)kvh * a.group) * HD + row_at(it.row0 + 16 * r + row);
                    *reinterpret_cast<float4 *>(dst + col) = make_float4(sum.x / ls, sum.y / ls, sum.z / ls, sum.w / ls);
                } else {
                    float *slab = a.part + (size_t)(it.part + kvh * R + r) * slab_floats(HD);
                    *reinterpret_cast<float4 *>(slab + row * HD + col) = sum;
                    if (col == 0) *reinterpret_cast<float2 *>(slab + 16 * HD + 2 * row) = make_float2(ms, ls);
                }
            }
            __syncthreads();
        }
        __syncthreads();  // lds and stat are written again
    }
}

// Joins a split tile's parts: a block a row, its waves over the parts.
template <int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
    constexpr int E = HD / 64;
    __shared__ float red[4][HD], stat[4][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // Rows of a join: those of its tile, for each KV head. gridDim.x walks them.
    for (uint32_t j = blockIdx.y; j < a.b.head->n_joins; j += gridDim.y) {
        const JoinAt join = a.b.joins[j];
        const SeqAt seq = a.b.seqs[join.seq];
        const uint32_t rows = min(16 * join.slabs, seq.n_new * a.group - join.row0);
        for (uint32_t i = blockIdx.x; i < rows * a.n_kv_heads; i += gridDim.x) {
            const uint32_t row = i % rows, kvh = i / rows;
            const float *part = a.part + (size_t)(join.part + kvh * join.slabs + row / 16) * slab_floats(HD);
            const size_t step = (size_t)join.slabs * a.n_kv_heads * slab_floats(HD);
            float top = -INFINITY, l = 0.f, acc[E];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
            for (uint32_t p = wave; p < join.n_parts; p += 4) {
                const float *s = part + p * step;
                const float2 ml = *reinterpret_cast<const float2 *>(s + 16 * HD + 2 * (row % 16));
                float x[E];
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = s[(row % 16) * HD + E * lane + e];
                const float now = fmaxf(top, ml.x);
                const float before = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - now);
                // A part of no weight has no maximum; one of NaN has none either.
                const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(ml.x - now);
                l = l * (top == -INFINITY && l != 0.f ? 1.f : before) + ml.y * f;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = fmaf(x[e], f, acc[e] * before);
                top = now;
            }
            if (lane == 0) {
                stat[wave][0] = top;
                stat[wave][1] = l;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) red[wave][E * lane + e] = acc[e];
            __syncthreads();
            if (threadIdx.x < HD) {
                const float all = fmaxf(fmaxf(stat[0][0], stat[1][0]), fmaxf(stat[2][0], stat[3][0]));
                float sum = 0.f, ls = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float f = stat[w][0] == -INFINITY ? (stat[w][1] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(stat[w][0] - all);
                    sum = fmaf(red[w][threadIdx.x], f, sum);
                    ls = fmaf(stat[w][1], f, ls);
                }
                const uint32_t r = join.row0 + row;
                a.out[((size_t)(seq.token0 + r / a.group) * a.n_heads + (size_t)kvh * a.group + r % a.group) * HD + threadIdx.x] = sum / ls;
            }
            __syncthreads();
        }
    }
}

// A captured launch's grid, whatever is set later: its blocks walk the items.
constexpr unsigned kCapturedBlocks = 1024;

template <int HD, int R>
hipError_t few(hipStream_t s, const PagedAttnArgs &a, int cls, unsigned grid, bool bf16) {
    if (bf16) paged_few_kernel<HD, R, uint16_t><<<grid, kFewThreads, 0, s>>>(a, cls);
    else paged_few_kernel<HD, R, float><<<grid, kFewThreads, 0, s>>>(a, cls);
    return hipGetLastError();
}

template <int HD>
hipError_t attention(hipStream_t s, const PagedAttnArgs &a, const BatchHead &count, bool bf16, bool captured) {
    for (int c = 0; c < kClasses; ++c) {
        const size_t items = (size_t)(count.first[c + 1] - count.first[c]) * a.n_kv_heads;
        if (!items && !(captured && c == 0)) continue;
        const unsigned grid = captured ? kCapturedBlocks : (unsigned)std::min<size_t>(items, 0x7fffffu);
        hipError_t e = hipSuccess;
        if (c == 0) e = few<HD, 1>(s, a, c, grid, bf16);
        if constexpr (HD < 256) {
            if (c == 1) e = few<HD, 2>(s, a, c, grid, bf16);
            if (c == 2) e = few<HD, 4>(s, a, c, grid, bf16);
        }
        if (e != hipSuccess) return e;
    }
    if (!count.n_joins && !captured) return hipSuccess;
    const dim3 grid = captured ? dim3(64, 64) : dim3(std::min(count.join_rows * a.n_kv_heads, 4096u), std::min(count.n_joins, 4096u));
    paged_join_kernel<HD><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_attention(hipStream_t s, const PagedAttnArgs &a, const BatchHead &count, size_t head_dim, bool bf16,
                                  bool captured) {
    if (count.n_tokens == 0 && !captured) return hipSuccess;
    return head_dim == 64    ? attention<64>(s, a, count, bf16, captured)
           : head_dim == 128 ? attention<128>(s, a, count, bf16, captured)
                             : attention<256>(s, a, count, bf16, captured);
}

}  // namespace th

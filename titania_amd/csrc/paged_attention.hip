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

// A class's items: as they are set, or, of a captured launch, as the head says.
struct Launch {
    uint32_t first, n;
    int cls;
    bool captured;
};

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

// What an earlier launch left and this one only reads, through the scalar cache.
template <typename T>
__device__ __forceinline__ T scalar_load(const T *p, size_t i) {
    T v;
    const auto *w = (const __attribute__((address_space(4))) uint32_t *)(uintptr_t)(p + i);
    uint32_t u[sizeof(T) / 4];
#pragma unroll
    for (size_t k = 0; k < sizeof(T) / 4; ++k) u[k] = w[k];
    __builtin_memcpy(&v, u, sizeof(T));
    return v;
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

// Tiles of up to 16 rows. Each of four waves takes 16 of every 64 positions
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
// A step's 64 products of 32 cycles take a wave 2048 cycles, while the block's
// 64 KB of f32 keys and values take a CU's share of HBM 8000: 16 rows cost what
// one costs. (With more sets of 16 a wave, 17 to 64 rows took 1.3 to 1.7 times
// what the kernel for many rows takes for them.)
//
// Bound by HBM: one token at 32767, 16 / 8 heads, f32, 53.5 us with the join
// (268 MB at 5.0 TB/s); 64 tokens at 120 to 8000, 32 / 8 heads, bf16, 202 us
// (5.3 TB/s). One token at 40 takes 5.8 us: a launch, the item, its page, its
// rows and two chains of products, each of which waits for the one before.
template <int HD, typename KV>
__global__ __launch_bounds__(kFewThreads, HD < 256 ? 2 : 1) void paged_few_kernel(PagedAttnArgs a, Launch launch) {
    constexpr int VE = 16 / sizeof(KV);         // values of 16 bytes
    constexpr int KJ = HD / (4 * VE);           // 16-byte loads of a lane's part of a key
    constexpr int VV = VE <= HD / 16 ? VE : HD / 16;  // values of a load of a value row, which 16 lanes share
    constexpr int VJ = HD / (16 * VV);          // such loads
    using VLoad = std::conditional_t<VV == VE, th_u32x4, u32x2>;
    constexpr int QS = HD + 4;                  // floats between rows in LDS
    constexpr int kMerge = 4 * 16 * (HD + 4);   // the waves' results of 16 rows
    __shared__ __align__(16) float lds[kMerge];
    __shared__ float stat[4][16][2];
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t first = launch.first, n = launch.n;
    if (launch.captured) {
        first = scalar_load(a.b.head->first, launch.cls);
        n = scalar_load(a.b.head->first, launch.cls + 1) - first;
    }
    n *= a.n_kv_heads;
    const float c2 = a.scale * kLog2e;
    for (uint32_t at = blockIdx.x; at < n; at += gridDim.x) {
        const ItemAt it = scalar_load(a.b.items, first + at / a.n_kv_heads);
        const int kvh = at % a.n_kv_heads;
        const SeqAt &seq = it.seq;
        const uint32_t rows = min(16u, seq.n_new * a.group - it.row0);
        const float *const qb = a.q + ((size_t)seq.token0 * a.n_heads + (size_t)kvh * a.group) * HD;
        // Row `row` of the sequence, in q and out.
        auto row_at = [&](uint32_t row) { return ((size_t)(row / a.group) * a.n_heads + row % a.group) * HD; };
        // Rows past the last repeat it. (Through LDS, to be read from memory once a
        // block, they would wait for each other's loads.)
        const uint32_t own = it.row0 + min((uint32_t)m, rows - 1), token = own / a.group;
        float q[KJ][VE];
        {
            const float *const qr = qb + row_at(own) + g * VE;
#pragma unroll
            for (int j = 0; j < KJ; ++j)
#pragma unroll
                for (int e = 0; e < VE; e += 4)
                    *reinterpret_cast<float4 *>(&q[j][e]) = *reinterpret_cast<const float4 *>(qr + j * 4 * VE + e);
        }
        const uint32_t *const pages = a.b.pages + seq.page0;
        const uint32_t mask = (1u << a.b.page_shift) - 1;
        // 16 positions from c on, a multiple of 16, lie in one page.
        auto page_of = [&](uint32_t c) { return scalar_load(pages, min(c, it.k1 - 1) >> a.b.page_shift); };
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
        f32x4 o[HD / 16];
        float mx = -INFINITY, l = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
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
            f32x4 s{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < KJ; ++j)
#pragma unroll
                for (int e = 0; e < VE; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j][e], q[j][e], s, 0, 0, 0);
            float x[4], top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = s[i] * c2;
            uint32_t seen = 0xffff;
            if (partly) {
                seen = seen16(seq, a.b.tree, token, c) & (it.k1 - c < 16 ? (1u << (it.k1 - c)) - 1 : 0xffffu);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = seen >> (4 * g + i) & 1 ? x[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max_nn(top, x[i]);
            top = max_nn(mx, rows_max_nn(top));
            const float base = top == -INFINITY ? 0.f : top;
            if (__any(top != mx)) {
                const float alpha = __builtin_amdgcn_exp2f(mx - base);
                l *= alpha;
#pragma unroll
                for (int d = 0; d < HD / 16; ++d) o[d] *= alpha;
                mx = top;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = __builtin_amdgcn_exp2f(x[i] - base);
                l += s[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int d = 0; d < HD / 16; ++d)
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[i][d / VV][d % VV], s[i], o[d], 0, 0, 0);
            // Values that are no numbers, which the products left out: for the
            // rows that see them alone.
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
                            if (!finite(f)) o[d][i] = fmaf(p, f, o[d][i]);
                        }
                }
            }
        }
        // The four waves' results: o[d][i] is dimension (d / VV) 16 VV +
        // (4 g + i) VV + d % VV of row m.
        l = rows_sum(l);
        if (g == 0) {
            stat[wave][m][0] = mx;
            stat[wave][m][1] = l;
        }
        __syncthreads();
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[w][m][0]);
        const float f = mx == -INFINITY ? (l == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(mx - top);
#pragma unroll
        for (int d = 0; d < HD / 16; d += 4)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4 *>(&lds[(wave * 16 + m) * QS + (d / VV) * 16 * VV + (4 * g + i) * VV + d % VV]) =
                    make_float4(o[d][i] * f, o[d + 1][i] * f, o[d + 2][i] * f, o[d + 3][i] * f);
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < rows * (HD / 4); i += kFewThreads) {
            const uint32_t row = i / (HD / 4), col = 4 * (i % (HD / 4));
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            float ms = -INFINITY, ls = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) ms = fmaxf(ms, stat[w][row][0]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float4 x = *reinterpret_cast<const float4 *>(&lds[(w * 16 + row) * QS + col]);
                sum = make_float4(sum.x + x.x, sum.y + x.y, sum.z + x.z, sum.w + x.w);
                const float mw = stat[w][row][0], lw = stat[w][row][1];
                ls += mw == -INFINITY ? lw : lw * __builtin_amdgcn_exp2f(mw - ms);
            }
            if (it.part == kNoPart) {
                float *dst = a.out + ((size_t)seq.token0 * a.n_heads + (size_t)kvh * a.group) * HD + row_at(it.row0 + row);
                *reinterpret_cast<float4 *>(dst + col) = make_float4(sum.x / ls, sum.y / ls, sum.z / ls, sum.w / ls);
            } else {
                float *slab = a.part + (size_t)(it.part + kvh) * slab_floats(HD);
                const float f = ls == 0.f ? 1.f : 1.f / ls;  // (zero: the row sees nothing here)
                *reinterpret_cast<float4 *>(slab + row * HD + col) = make_float4(sum.x * f, sum.y * f, sum.z * f, sum.w * f);
                if (col == 0) *reinterpret_cast<float2 *>(slab + 16 * HD + 2 * row) = make_float2(ms, ls);
            }
        }
        __syncthreads();  // lds and stat are written again
    }
}

// ---- tiles of many rows ----

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kManyThreads = 512, kManyKeys = 64;

// Two f32 as f16 terms hi + lo, each to the nearest: 22 bits of a value within
// 2^16 below the largest that f16 holds, 2^-25 below that of any.
template <bool LO>
__device__ __forceinline__ void split_f16(float a, float b, uint32_t &hi, uint32_t &lo) {
    const f16x2 h = __builtin_convertvector((f32x2){a, b}, f16x2);
    hi = __builtin_bit_cast(uint32_t, h);
    if constexpr (LO) {  // what is left, exactly, in an instruction that takes the f16 as it is
        float c, d;
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(c) : "v"(hi), "v"(a));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(hi), "v"(b));
        lo = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){c, d}, f16x2));
    }
}

// The larger; NaN if one is (three of them are one instruction).
__device__ __forceinline__ float max_or_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7fffffffu; }
// The exponent that brings values of at most this magnitude below 2^15.
__device__ __forceinline__ int shift_of(uint32_t most) { return 14 + 127 - (int)(most >> 23); }

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false));
}
// The maximum over each 16 lanes, in each of them.
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = dpp_max<0xB1>(v);          // quad_perm [1,0,3,2]
    v = dpp_max<0x4E>(v);          // quad_perm [2,3,0,1]
    v = dpp_max<0x124>(v);         // row_ror:4
    return dpp_max<0x128>(v);      // row_ror:8
}
// Over the lanes that are a multiple of 16 apart, in each of them.
__device__ __forceinline__ uint32_t across_max(uint32_t v) {
    auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(p[0], p[1]);
    auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(q[0], q[1]);
}

// Which of the 64 positions from c on a sequence's token sees.
__device__ __forceinline__ uint64_t seen64(const SeqAt &seq, const uint64_t *tree, uint32_t token, uint32_t c) {
    const int d = (int)(c - seq.context);
    const int before = d >= 0 ? 0 : d <= -64 ? 64 : -d;
    if (!seq.is_tree) {
        const int n = (int)token + 1 - d;
        return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
    }
    const uint64_t *words = tree + (size_t)(seq.token0 + token) * kTreeWords;
    const int at = d < 0 ? 0 : d, word = at >> 6, shift = at & 63;
    const uint64_t low = words[word] >> shift, high = words[word + 1 < kTreeWords ? word + 1 : word];
    const uint64_t bits = low | (shift && word + 1 < kTreeWords ? high << (64 - shift) : 0ull);
    return before == 64 ? ~0ull : (bits << before) | ((1ull << before) - 1);
}

// Tiles of up to 128 SETS rows: eight waves of SETS sets of 16, positions 64 at
// a time through LDS, in two buffers: while a tile's products run, the next
// one's keys and values, already in registers, are converted and stored, and
// the one after it is requested. One barrier a tile.
//
// Products on v_mfma_f32_16x16x32_f16, every f32 as two f16 terms and a product
// as hi hi + hi lo + lo hi (values of a bf16 cache are one f16 term, exactly,
// and two products). What f16 lacks in range powers of two make up: of each
// query row its own, of a tile's keys one, and of its values one, the smallest
// so far, to which a row's sums are brought along when it changes;
// the weights are of exp2(x - r + 10), r the row's maximum, or within
// 2^5 of it. Results are those of f32 but for
// 2^-21 of a product, and for what lies 2^38 below the largest value that a
// row sees, or 2^25 below where unseen ones are larger (by 2^13 at most, as follows).
//
// S^T = K Q^T leaves a lane four neighbouring positions of its row in each of
// the tile's four sixteens, which with V^T's columns in that order are the
// operand of O^T = V^T P^T.
//
// Where a tile has an infinity or a NaN, or where not all of the item's rows see
// all positions and these differ by more than 2^12 (of a tree's values, over its
// tiles so far: a row may see none of an earlier tile whose scale is its own
// tile's), the item is done again from memory, in f32, a position at a time and
// each row for itself: what it does not see does not reach it. (These are no
// numbers to be fast with: a prompt of 2048 one of whose positions has 2^-14 of
// its neighbours' values takes 2.9 ms, not 0.14, for that position's own rows;
// 512 tokens at 8000 with an infinity in their context 11 ms, not 0.2.)
//
// Bound by the matrix and the vector units in turn: a wave's products wait for
// its conversions and its softmax, and a SIMD's two waves hide half of that from
// each other. Chunks of 2048, 1946 and 1592 tokens at 2500, 0 and 5000, 32 / 8
// heads, f32, take 0.81 ms, products at 1.1 PFLOP/s, the matrix units busy 51% of
// the time (a large matrix product of a library: 1.24 PFLOP/s). That case, step by step:
// f32 products 3.87 ms; two f16 terms 1.60; one exponent for a tile's keys and
// maxima by lane exchanges 1.12; rows swizzled in LDS, not padded, 1.07;
// remainders by one mixed-precision fma, maxima of three 0.98; references that
// move by 2^5 only 0.95; products before other waves' conversions 0.91; the
// longest items first 0.85; half of the waves converting between their halves
// of a tile 0.81 to 0.83; positions compared only where not all rows see them
// 0.81 (0.83 in the same minutes without). A tree of 60 tokens at 12001 takes 56 to 60
// us, 8.5 of them the join: 256 blocks of 6 tiles of 5.6 us, and 34 MB of
// partial results.
// Not kept: two groups of four waves that halve a tile's positions, for up to
// 64 rows (bf16 41 -> 44 us, f32 66 -> 63); two tiles requested ahead, or the
// first one before the queries are converted (no change); blocks' rows on turned
// waves, so that the few that have some share the SIMDs (no change).
template <int HD, int SETS, typename KV>
__global__ __launch_bounds__(kManyThreads, SETS == 1 && sizeof(KV) == 2 ? 4 : 2) void paged_many_kernel(PagedAttnArgs a, Launch launch) {
    constexpr bool F32 = sizeof(KV) == 4;
    constexpr int KT = kManyKeys, RW = 16 * SETS;
    constexpr bool kAhead = F32 || SETS > 1;
    constexpr float kGrow = 5.f, kBase = 10.f;  // weights below 2^15
    constexpr uint32_t KB = 2 * HD, VB = 2 * KT;  // bytes of a key, and of a dimension's positions
    constexpr int LPK = HD / 8;                // lanes a key
    constexpr int KU = KT * LPK / kManyThreads;  // keys' units (8 values) of a thread
    constexpr int VD = HD / 64;                // neighbouring dimensions of a thread, of 8 positions
    // A buffer's parts, in bytes: keys hi, lo, values hi, lo.
    constexpr uint32_t kKL = KT * KB, kVH = (F32 ? 2 : 1) * kKL, kVL = kVH + HD * VB, kBuf = F32 ? kVL + HD * VB : kVL;
    __shared__ __align__(16) char lds[2 * kBuf];
    __shared__ __align__(16) uint4 looked[2][8];  // of a wave's part of a tile: magnitudes, as below
    __shared__ uint32_t odd_of[4];
    const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t first = launch.first, n = launch.n;
    if (launch.captured) {
        first = scalar_load(a.b.head->first, launch.cls);
        n = scalar_load(a.b.head->first, launch.cls + 1) - first;
    }
    n *= a.n_kv_heads;
    const float c2 = a.scale * kLog2e;
    if (blockIdx.x >= n) return;
    const ItemAt it = scalar_load(a.b.items, first + blockIdx.x / a.n_kv_heads);
    const int kvh = blockIdx.x % a.n_kv_heads;
    const SeqAt &seq = it.seq;
    const uint32_t rows = min((uint32_t)(8 * RW), seq.n_new * a.group - it.row0);
    const int wrow = RW * wave;  // the wave's first row
    const size_t qbase = ((size_t)seq.token0 * a.n_heads + (size_t)kvh * a.group) * HD;
    auto row_at = [&](uint32_t row) { return qbase + ((size_t)(row / a.group) * a.n_heads + row % a.group) * HD; };
    uint32_t token[SETS];
    uint4 qh[SETS][HD / 32], ql[SETS][HD / 32];
    float qf[SETS];  // the scale of a row's scores, c2 in it
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
        const uint32_t row = it.row0 + min((uint32_t)(wrow + 16 * s + li), rows - 1);  // past the last: it again
        token[s] = row / a.group;
        const float *const src = a.q + row_at(row) + 8 * lg;
        float f[HD / 32][8];
        uint32_t most = 0;
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
            const float4 x = *reinterpret_cast<const float4 *>(src + 32 * c);
            const float4 y = *reinterpret_cast<const float4 *>(src + 32 * c + 4);
            const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[c][e] = v[e];
                most = max(most, magnitude(v[e]));
            }
        }
        most = across_max(most);
        const int sh = shift_of(most);
        qf[s] = ldexpf(c2, -sh);
#pragma unroll
        for (int c = 0; c < HD / 32; ++c) {
            uint32_t h[4], l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) split_f16<true>(ldexpf(f[c][2 * e], sh), ldexpf(f[c][2 * e + 1], sh), h[e], l[e]);
            qh[s][c] = make_uint4(h[0], h[1], h[2], h[3]);
            ql[s][c] = make_uint4(l[0], l[1], l[2], l[3]);
        }
    }
    // The first position that one of the item's rows does not see.
    const uint32_t in_common = seq.context + (seq.is_tree ? 0 : it.row0 / a.group + 1);
    // Of the wave's rows: the first position that one does not see, and the
    // first that none sees (zero: there are no such rows).
    const uint32_t w0 = wrow, w1 = min(w0 + RW, rows) - 1;
    const uint32_t all_see = seq.context + (seq.is_tree ? 0 : (it.row0 + min(w0, rows - 1)) / a.group + 1);
    const uint32_t none_sees = w0 >= rows ? 0 : seq.context + (it.row0 + w1) / a.group + 1;
    f32x4 o[SETS][HD / 16];
    float mx[SETS], l[SETS];
    int units[SETS];  // o is of values times 2^units
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
        mx[s] = -INFINITY;
        l[s] = 0.f;
        units[s] = 0;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) o[s][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const uint32_t *const pages = a.b.pages + seq.page0;
    const uint32_t mask = (1u << a.b.page_shift) - 1;
    const size_t to_v = ((size_t)a.n_kv_heads << a.b.page_shift) * HD;
    // A key's row, with its sixteen's page: positions past the last repeat its page.
    auto row_of = [&](uint32_t pos) {
        const size_t page = scalar_load(pages, min(pos, it.k1 - 1) >> a.b.page_shift);
        return static_cast<const KV *>(a.cache) +
               ((((page * 2 * a.n_kv_heads + kvh)) << a.b.page_shift) + (pos & mask)) * HD;
    };
    // What a thread stages: keys kkey + KT / KU i, 8 values from 8 kch;
    // values of dimensions VD lane + {0, ..}, of the 8 positions that are
    // operand group `wave`: sixteens 2 sigma and 2 sigma + 1, four of each.
    // (Formed from the thread's number where they are used: with all of them
    // kept, the registers do not suffice.)
    const int wkey = wave * (64 / LPK);  // the wave's first
    const int vkey = 32 * (wave >> 2) + 4 * (wave & 3);
    auto thread = [] {
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));
        return t;
    };
    // Where 16 bytes of a row lie: rows of 256 bytes cover the banks, two of
    // 128 do. What the lanes of a fragment's read take, and neighbouring
    // lanes write, is in as many banks.
    auto swizzled = [](uint32_t bytes, uint32_t row, uint32_t chunk) {
        return row * bytes + 16 * (chunk ^ (bytes == 256 ? row & 15 : row >> 1 & 7));
    };
    auto at_lds = [&](uint32_t o) -> uint4 & { return *reinterpret_cast<uint4 *>(lds + o); };
    float kraw[KU][8], vraw[8][VD];
    auto fetch = [&](uint32_t c0) {
        const int tid = thread();
        const uint32_t klane = ((tid / LPK - (wkey & ~15)) * HD + 8 * (tid % LPK)) * sizeof(KV);
        const uint32_t vlane = VD * (tid & 63) * sizeof(KV);
#pragma unroll
        for (int i = 0; i < KU; ++i) {
            const KV *src = reinterpret_cast<const KV *>(
                reinterpret_cast<const char *>(row_of(c0 + (wkey & ~15) + KT / KU * i)) + klane);
            if constexpr (F32) {
                const float4 x = *reinterpret_cast<const float4 *>(src), y = *reinterpret_cast<const float4 *>(src + 4);
                const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) kraw[i][e] = v[e];
            } else {
                const uint4 w = *reinterpret_cast<const uint4 *>(src);
                kraw[i][0] = __uint_as_float(w.x); kraw[i][1] = __uint_as_float(w.y);
                kraw[i][2] = __uint_as_float(w.z); kraw[i][3] = __uint_as_float(w.w);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const KV *src = reinterpret_cast<const KV *>(
                reinterpret_cast<const char *>(row_of(c0 + 32 * (wave >> 2) + 16 * h) + to_v + 4 * (wave & 3) * HD) + vlane);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (F32 && VD == 2) {
                    const float2 x = *reinterpret_cast<const float2 *>(src + j * HD);
                    vraw[4 * h + j][0] = x.x;
                    vraw[4 * h + j][1] = x.y;
                } else if constexpr (F32) {
                    vraw[4 * h + j][0] = src[j * HD];
                } else if constexpr (VD == 2) {
                    vraw[4 * h + j][0] = __uint_as_float(*reinterpret_cast<const uint32_t *>(src + j * HD));
                } else {
                    vraw[4 * h + j][0] = __uint_as_float((uint32_t)src[j * HD]);
                }
            }
        }
    };
    // As f32 from what is in registers.
    auto value = [&](int j, int d) {
        if constexpr (F32) return vraw[j][d];
        else return d ? bf16_hi(__float_as_uint(vraw[j][0])) : bf16_lo(__float_as_uint(vraw[j][0]));
    };
    auto key_value = [&](int i, int e) {
        if constexpr (F32) return kraw[i][e];
        else return e & 1 ? bf16_hi(__float_as_uint(kraw[i][e / 2])) : bf16_lo(__float_as_uint(kraw[i][e / 2]));
    };
    // The largest magnitude of the wave's keys and values, and, where some
    // row does not see some position, the smallest of a position's largest
    // (which takes lane exchanges for each: wherever a position was new, a
    // prompt of 2048 from its start took 151 us, not 136).
    auto look = [&](uint32_t c0, uint32_t tile) {
        uint32_t ktop = 0, vtop = 0, kleast = 0x7f000000u, vleast = 0x7f000000u;
        if (c0 + KT > it.k1) {  // past the last position is anything: zero
            const int tid = thread();
#pragma unroll
            for (int i = 0; i < KU; ++i)
#pragma unroll
                for (int e = 0; e < (F32 ? 8 : 4); ++e)
                    kraw[i][e] = c0 + tid / LPK + KT / KU * i < it.k1 ? kraw[i][e] : 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int d = 0; d < (F32 ? VD : 1); ++d)
                    vraw[j][d] = c0 + vkey + (j & 3) + 16 * (j >> 2) < it.k1 ? vraw[j][d] : 0.f;
        }
        if (c0 + KT > in_common) {
#pragma unroll
            for (int i = 0; i < KU; ++i) {
                uint32_t own = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) own = max(own, magnitude(key_value(i, e)));
                own = LPK == 16 ? row_max(own) : dpp_max<0x141>(dpp_max<0x4E>(dpp_max<0xB1>(own)));  // row_half_mirror
                ktop = max(ktop, own);
                kleast = own ? min(kleast, own) : kleast;
            }
            kleast = ~across_max(row_max(~kleast));
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                uint32_t own = 0;
#pragma unroll
                for (int d = 0; d < VD; ++d) own = max(own, magnitude(value(j, d)));
                own = across_max(row_max(own));
                vtop = max(vtop, own);
                vleast = own ? min(vleast, own) : vleast;
            }
            ktop = across_max(row_max(ktop));
        } else {
            float k = 0.f, v = 0.f;
#pragma unroll
            for (int i = 0; i < KU; ++i)
#pragma unroll
                for (int e = 0; e < 8; e += 2)
                    k = max_or_nan(max_or_nan(k, __builtin_fabsf(key_value(i, e))), __builtin_fabsf(key_value(i, e + 1)));
#pragma unroll
            for (int j = 0; j < 8; j += 2)
#pragma unroll
                for (int d = 0; d < VD; ++d)
                    v = max_or_nan(max_or_nan(v, __builtin_fabsf(value(j, d))), __builtin_fabsf(value(j + 1, d)));
            ktop = across_max(row_max(magnitude(k)));
            vtop = across_max(row_max(magnitude(v)));
        }
        if ((thread() & 63) == 0) looked[tile & 1][wave] = make_uint4(ktop, vtop, kleast, vleast);
    };
    int shift = 1 << 20;  // of the last tile's values; at first more than any
    int kshift = 0;       // of the last tile's keys
    // The largest magnitude of a tree's values behind its context so far, of
    // which a row may see none while its own are scaled with it.
    uint32_t drafted = 0;
    // The tile in registers to LDS.
    auto store = [&](uint32_t tile) {
        // A wave's part a lane, the eight of them over each 16 lanes.
        const int tid = thread(), kkey = tid / LPK, kch = tid % LPK;
        const uint4 w = looked[tile & 1][tid & 7];
        auto uniform_max = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)row_max(v)); };
        const uint32_t ktop = uniform_max(w.x), vtop = uniform_max(w.y), kleast = ~uniform_max(~w.z), vleast = ~uniform_max(~w.w);
        const bool branches = seq.is_tree && it.k0 + (tile + 1) * KT > in_common;
        if (branches) drafted = max(drafted, vtop);
        const uint32_t vmost = branches ? drafted : vtop;
        // Infinities and NaN; positions 2^12 apart that not all rows see, whose
        // values have a scale in common also over a tree's tiles.
        const bool odd = max(ktop, vtop) >= 0x7f800000u || (kleast < ktop && (ktop >> 23) - (kleast >> 23) > 12) ||
                         (vleast < vmost && (vmost >> 23) - (vleast >> 23) > 12);
        if (!odd) shift = min(shift, shift_of(vtop));
        kshift = shift_of(ktop);
        const uint32_t buf = (tile & 1) * kBuf;
        const uint32_t kput = buf + swizzled(KB, kkey, kch);
#pragma unroll
        for (int i = 0; i < KU; ++i) {
            uint32_t h[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                split_f16<F32>(ldexpf(key_value(i, 2 * e), kshift), ldexpf(key_value(i, 2 * e + 1), kshift), h[e], lo[e]);
            const uint32_t to = kput + KT / KU * i * KB;
            at_lds(to) = make_uint4(h[0], h[1], h[2], h[3]);
            if constexpr (F32) at_lds(to + kKL) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
#pragma unroll
        for (int d = 0; d < VD; ++d) {
            uint32_t h[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                split_f16<F32>(ldexpf(value(2 * e, d), shift), ldexpf(value(2 * e + 1, d), shift), h[e], lo[e]);
            const uint32_t to = buf + kVH + swizzled(VB, VD * (tid & 63) + d, wave);
            at_lds(to) = make_uint4(h[0], h[1], h[2], h[3]);
            if constexpr (F32) at_lds(to + kVL - kVH) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        if (odd) odd_of[tile & 3] = 1;
    };
    // Scores, weights and sums of 32 positions at a time (of 64: 16 more
    // registers for scores and 16 for weights than there are).
    auto products = [&](int h, uint32_t c0, uint32_t tile, int tile_shift, int tile_kshift) {
        auto mfma = [](const uint4 &x, const uint4 &y, const f32x4 &z) {
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), z, 0, 0, 0);
        };
        const bool masked = c0 + KT > all_see || c0 + KT > it.k1;
        const int tid = thread(), li = tid & 15, lg = tid >> 4 & 3;
        const uint32_t buf = (tile & 1) * kBuf, kget = buf + swizzled(KB, li, lg), vget = buf + kVH + swizzled(VB, li, lg);
        {
            f32x4 st[SETS][2];
#pragma unroll
            for (int s = 0; s < SETS; ++s)
#pragma unroll
                for (int j = 0; j < 2; ++j) st[s][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            const uint32_t vb = vget ^ 64 * h;  // the chunk 4 h + lg
            // A step's fragments are requested before the products of the
            // one before it (where there are registers for both).
            uint4 x[2][2], y[2][F32 ? 2 : 1];
            auto key_fragments = [&](int c) {
                const uint32_t kb = (kget ^ 64 * c) + 32 * h * KB;  // the chunk 4 c + lg
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    x[c & 1][j] = at_lds(kb + 16 * j * KB);
                    if constexpr (F32) y[c & 1][j] = at_lds(kb + kKL + 16 * j * KB);
                }
            };
            if (kAhead) key_fragments(0);
            __builtin_amdgcn_s_setprio(1);  // products before another wave's conversions
#pragma unroll
            for (int c = 0; c < HD / 32; ++c) {
                if (!kAhead) key_fragments(c);
                else if (c + 1 < HD / 32) key_fragments(c + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int s = 0; s < SETS; ++s)
#pragma unroll
                    for (int j = 0; j < 2; ++j) st[s][j] = mfma(x[c & 1][j], qh[s][c], st[s][j]);
#pragma unroll
                for (int s = 0; s < SETS; ++s)
#pragma unroll
                    for (int j = 0; j < 2; ++j) st[s][j] = mfma(x[c & 1][j], ql[s][c], st[s][j]);
                if constexpr (F32)
#pragma unroll
                    for (int s = 0; s < SETS; ++s)
#pragma unroll
                        for (int j = 0; j < 2; ++j) st[s][j] = mfma(y[c & 1][j], qh[s][c], st[s][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
            uint4 ph[SETS], pl[SETS];
#pragma unroll
            for (int s = 0; s < SETS; ++s) {
                if (masked) {
                    uint32_t own = token[s];
                    asm volatile("" : "+v"(own));  // (nothing of it formed ahead)
                    uint64_t all = seen64(seq, a.b.tree, own, c0);
                    if (it.k1 - c0 < 64) all &= (1ull << (it.k1 - c0)) - 1;
                    const uint32_t seen = (uint32_t)(all >> 32 * h) >> 4 * lg;
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) st[s][j][e] = seen >> (16 * j + e) & 1 ? st[s][j][e] : -INFINITY;
                }
                float top = -INFINITY;
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; e += 2) top = max_or_nan(max_or_nan(top, st[s][j][e]), st[s][j][e + 1]);
                // Scores in units of log2. (Neither zero nor infinite: what is
                // not seen is -inf, and stays it.)
                const float f = fminf(fmaxf(ldexpf(qf[s], -tile_kshift), 0x1p-126f), 0x1p127f);
                top = rows_max_nn(top) * f;
                const bool any = top != -INFINITY;  // the row sees some
                // The reference moves when the maximum is 2^kGrow past it.
                if (__any(top > mx[s] + kGrow || (any && units[s] != tile_shift))) {
                    const float next = max_nn(mx[s], top);
                    const float alpha = mx[s] == next ? 1.f : __builtin_amdgcn_exp2f(mx[s] - next);
                    mx[s] = next;
                    l[s] *= alpha;
                    const int by = any ? tile_shift - units[s] : 0;
                    units[s] += by;
                    const float g = ldexpf(alpha, by);
#pragma unroll
                    for (int d = 0; d < HD / 16; ++d) o[s][d] *= g;
                }
                const float base = mx[s] == -INFINITY ? 0.f : kBase - mx[s];
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        st[s][j][e] = __builtin_amdgcn_exp2f(fmaf(st[s][j][e], f, base));
                        l[s] += st[s][j][e];
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    split_f16<true>(st[s][e / 2][2 * (e & 1)], st[s][e / 2][2 * (e & 1) + 1], hi[e], lo[e]);
                ph[s] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                pl[s] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            auto value_fragments = [&](int n) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    x[n & 1][i] = at_lds(vb + 16 * (2 * n + i) * VB);
                    if constexpr (F32) y[n & 1][i] = at_lds(vb + kVL - kVH + 16 * (2 * n + i) * VB);
                }
            };
            if (kAhead) value_fragments(0);
#pragma unroll
            for (int n = 0; n < HD / 32; ++n) {
                if (!kAhead) value_fragments(n);
                else if (n + 1 < HD / 32) value_fragments(n + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int s = 0; s < SETS; ++s)
#pragma unroll
                    for (int i = 0; i < 2; ++i) o[s][2 * n + i] = mfma(x[n & 1][i], ph[s], o[s][2 * n + i]);
#pragma unroll
                for (int s = 0; s < SETS; ++s)
#pragma unroll
                    for (int i = 0; i < 2; ++i) o[s][2 * n + i] = mfma(x[n & 1][i], pl[s], o[s][2 * n + i]);
                if constexpr (F32)
#pragma unroll
                    for (int s = 0; s < SETS; ++s)
#pragma unroll
                        for (int i = 0; i < 2; ++i) o[s][2 * n + i] = mfma(y[n & 1][i], ph[s], o[s][2 * n + i]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    // A row set's results, or partial ones: x[d][e] 2^-by is dimension
    // 16 d + 4 lg + e of the lane's row, of weights exp2(. - top) that add up
    // to `sum` (2^15 for each position at most: over them first).
    auto put = [&](int s, const f32x4 (&x)[HD / 16], float top, float sum, int by) {
        const int tid = thread(), li = tid & 15, g4 = 4 * (tid >> 4 & 3);
        const uint32_t r = wrow + 16 * s + li;
        if (r >= rows) return;
        float *dst;
        float f = 1.f / sum;
        if (it.part == kNoPart) {
            dst = a.out + row_at(it.row0 + r);
        } else {
            dst = a.part + (size_t)(it.part + kvh * 8 * SETS + r / 16) * slab_floats(HD);
            if (sum == 0.f) f = 1.f;  // it sees nothing here
            if (g4 == 0) *reinterpret_cast<float2 *>(dst + 16 * HD + 2 * li) = make_float2(top, sum);
            dst += li * HD;
        }
#pragma unroll
        for (int d = 0; d < HD / 16; ++d)
            *reinterpret_cast<float4 *>(dst + 16 * d + g4) = make_float4(ldexpf(x[d][0] * f, -by), ldexpf(x[d][1] * f, -by),
                                                                        ldexpf(x[d][2] * f, -by), ldexpf(x[d][3] * f, -by));
    };
    // A row set from memory, from the first position on, one at a time.
    auto one_by_one = [&](int s) {
        auto as_f32 = [](KV w) { return F32 ? (float)w : bf16_to_f32((uint16_t)w); };
        const int own = thread() & 63, g4 = 4 * (own >> 4);
        const uint32_t row = it.row0 + min((uint32_t)(wrow + 16 * s + (own & 15)), rows - 1);
        const float *const qr = a.q + row_at(row) + g4;
        f32x4 x[HD / 16];
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) x[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (uint32_t key = it.k0; key < it.k1; ++key) {
            const KV *const kr = row_of(key) + g4, *const vr = kr + to_v;
            float y = 0.f;
#pragma unroll 2
            for (int d = 0; d < HD / 16; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) y = fmaf(qr[16 * d + e], as_f32(kr[16 * d + e]), y);
            y = rows_sum(y) * c2;
            const bool sees = seen64(seq, a.b.tree, row / a.group, key) & 1;
            y = sees ? y : -INFINITY;
            const float next = max_nn(top, y), base = next == -INFINITY ? 0.f : next;
            const float alpha = top == -INFINITY ? (sum == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(top - base);
            const float p = __builtin_amdgcn_exp2f(y - base);
            top = next;
            sum = sum * alpha + p;
#pragma unroll
            for (int d = 0; d < HD / 16; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float more = fmaf(p, as_f32(vr[16 * d + e]), x[d][e] * alpha);
                    x[d][e] = sees ? more : x[d][e];
                }
        }
        put(s, x, top, sum, 0);
    };
    const uint32_t tiles = (it.k1 - it.k0 + KT - 1) / KT;
    if (threadIdx.x < 4) odd_of[threadIdx.x] = 0;
    fetch(it.k0);
    look(it.k0, 0);
    __syncthreads();
    store(0);
    int now = shift, know = kshift;
    if (tiles > 1) fetch(it.k0 + KT);
    uint32_t t = 0;
    for (; t < tiles; ++t) {
        const uint32_t c0 = it.k0 + t * KT;
        if (t + 1 < tiles) look(c0 + KT, t + 1);
        __syncthreads();  // tile t is stored, the other buffer free, the next one looked at
        if (odd_of[t & 3]) break;
        if (threadIdx.x == 0) odd_of[(t + 3) & 3] = 0;  // tile t - 1's, for tile t + 3
        auto next = [&] {
            if (t + 1 < tiles) store(t + 1);
            if (t + 2 < tiles) fetch(c0 + 2 * KT);
        };
        if (wave < 4) next();
        if (c0 < none_sees) products(0, c0, t, now, know);
        if (wave >= 4) next();
        if (c0 < none_sees) products(1, c0, t, now, know);
        now = shift;
        know = kshift;
    }
    if (none_sees) {
        if (__builtin_expect(t < tiles, 0)) {
#pragma unroll
            for (int s = 0; s < SETS; ++s) one_by_one(s);
        } else {
#pragma unroll
            for (int s = 0; s < SETS; ++s) put(s, o[s], mx[s] - kBase, rows_sum(l[s]), units[s]);
        }
    }
}

// Joins a split tile's parts, `W` waves a row: four for few rows of many parts,
// which then wait for a quarter of them, one for many rows (1920 rows of 32
// parts, 32 MB, 8.5 us; 16 rows of 64 parts 4.9). A part counts for its share of
// the weights: no sum here is larger than the values.
template <int HD, int W>
__device__ __forceinline__ void join_rows(const PagedAttnArgs &a, const BatchHead &head) {
    constexpr int E = HD / 64, ROWS = 4 / W;  // a block's rows
    __shared__ float red[W == 1 ? 1 : 4][W == 1 ? 1 : HD];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // gridDim.y walks the tiles, gridDim.x their rows, for each KV head.
    for (uint32_t j = blockIdx.y; j < head.n_joins; j += gridDim.y) {
        const JoinAt join = scalar_load(a.b.joins, j);
        const uint32_t rows = join.rows, n = join.n_parts;
        for (uint32_t i = blockIdx.x * ROWS + (W == 1 ? wave : 0); i < rows * a.n_kv_heads; i += gridDim.x * ROWS) {
            const uint32_t row = i % rows, kvh = i / rows;
            const float *const part = a.part + (size_t)(join.part + kvh * join.slabs + row / 16) * slab_floats(HD);
            const size_t step = (size_t)join.slabs * a.n_kv_heads * slab_floats(HD);
            auto stat = [&](uint32_t p) {
                return *reinterpret_cast<const float2 *>(part + p * step + 16 * HD + 2 * (row % 16));
            };
            auto fetch = [&](float (&x)[E], uint32_t p) {
                const float *s = part + p * step + (row % 16) * HD + E * lane;
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = s[e];
            };
            // The maximum and the sum of all parts, a part a lane; with one wave a
            // row, while the first parts are on their way.
            const float2 mine = lane < (int)n ? stat(lane) : make_float2(-INFINITY, 0.f);
            float ahead[W == 1 ? 8 : 1][E];
            auto fetch8 = [&](uint32_t p) {
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k)
                    if (p + k < n) fetch(ahead[k], p + k);
            };
            if constexpr (W == 1) fetch8(0);
            float top = mine.x, acc[E];
            for (uint32_t p = 64 + lane; p < n; p += 64) top = fmaxf(top, stat(p).x);
            top = wave_max_dpp(top);
            // A part's weights, by the largest of all: none where it has no
            // maximum, unless they are NaN.
            auto weight = [&](const float2 &ml) { return ml.y * __builtin_amdgcn_exp2f(ml.x - top); };
            float l = weight(mine);
            for (uint32_t p = 64 + lane; p < n; p += 64) l += weight(stat(p));
            const float over = 1.f / wave_sum_dpp(l);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = 0.f;
            auto add = [&](const float (&x)[E], float f) {
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = fmaf(x[e], f, acc[e]);
            };
            if constexpr (W == 1) {
                for (uint32_t p = 0; p < n; p += 8) {
                    if (p) fetch8(p);
                    const float share = (p < 64 ? weight(mine) : weight(stat(min((p & ~63u) + lane, n - 1)))) * over;
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k)
                        if (p + k < n)
                            add(ahead[k], __int_as_float(__builtin_amdgcn_readlane(__float_as_int(share), (p + k) & 63)));
                }
            } else {
#pragma unroll 8
                for (uint32_t p = wave; p < n; p += W) {
                    float x[E];
                    fetch(x, p);
                    add(x, weight(stat(p)) * over);
                }
            }
            const uint32_t r = join.row0 + row;
            float *out = a.out + ((size_t)(join.token0 + r / a.group) * a.n_heads + (size_t)kvh * a.group + r % a.group) * HD;
            if constexpr (W == 1) {
#pragma unroll
                for (int e = 0; e < E; ++e) out[E * lane + e] = acc[e];
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) red[wave][E * lane + e] = acc[e];
                __syncthreads();
                if (threadIdx.x < HD)
                    out[threadIdx.x] = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
                __syncthreads();
            }
        }
    }
}

constexpr uint32_t kManyRows = 2048;  // of a join's launch

// (Which of the two goes by the plan alone: a captured launch gives the bits of
// any other.)
template <int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
    const BatchHead head = scalar_load(a.b.head, 0);
    if (head.join_rows * a.n_kv_heads * head.n_joins > kManyRows) join_rows<HD, 1>(a, head);
    else join_rows<HD, 4>(a, head);
}

// A captured launch's grid, whatever is set later: the few-row kernel's blocks
// walk the items, the others' have one each, of the most that there can be: a
// sequence has 17 rows at least, a whole tile 128, and the rounds bound the splits.
constexpr unsigned kCapturedBlocks = 1024;
unsigned captured_blocks(const PagedAttnArgs &a, const BatchHead &count) {
    const size_t rows = (size_t)count.n_tokens * a.group;
    return (unsigned)((rows / 17 + rows / 128 + 2) * a.n_kv_heads + kMostSplitBlocks);
}

template <int HD>
hipError_t few(hipStream_t s, const PagedAttnArgs &a, const Launch &l, unsigned grid, bool bf16) {
    if (bf16) paged_few_kernel<HD, uint16_t><<<grid, kFewThreads, 0, s>>>(a, l);
    else paged_few_kernel<HD, float><<<grid, kFewThreads, 0, s>>>(a, l);
    return hipGetLastError();
}

template <int HD, int SETS>
hipError_t many(hipStream_t s, const PagedAttnArgs &a, const Launch &l, unsigned grid, bool bf16) {
    if (bf16) paged_many_kernel<HD, SETS, uint16_t><<<grid, kManyThreads, 0, s>>>(a, l);
    else paged_many_kernel<HD, SETS, float><<<grid, kManyThreads, 0, s>>>(a, l);
    return hipGetLastError();
}

template <int HD>
hipError_t attention(hipStream_t s, const PagedAttnArgs &a, const BatchHead &count, bool bf16, unsigned captured) {
    for (int c = 0; c < kClasses; ++c) {
        const Launch l{count.first[c], count.first[c + 1] - count.first[c], c, captured != 0};
        const size_t blocks = (size_t)l.n * a.n_kv_heads;
        if (!blocks && !(captured >> c & 1)) continue;
        // (The few-row kernel's blocks walk the items past 2^22, too.)
        const unsigned grid = c == 0 ? (unsigned)std::min<size_t>(captured ? kCapturedBlocks : blocks, (size_t)1 << 22)
                                     : captured ? captured_blocks(a, count) : (unsigned)blocks;
        hipError_t e = hipSuccess;
        if (c == 0) e = few<HD>(s, a, l, grid, bf16);
        if constexpr (HD < 256) {
            if (c == 1) e = many<HD, 1>(s, a, l, grid, bf16);
            if (c == 2) e = many<HD, 2>(s, a, l, grid, bf16);
        }
        if (e != hipSuccess) return e;
    }
    if (!count.n_joins && !captured) return hipSuccess;
    const uint32_t rows = count.join_rows * a.n_kv_heads, blocks = rows * count.n_joins > kManyRows ? (rows + 3) / 4 : rows;
    const dim3 grid = captured ? dim3(64, 64) : dim3(std::min(blocks, 4096u), std::min(count.n_joins, 4096u));
    paged_join_kernel<HD><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_attention(hipStream_t s, const PagedAttnArgs &a, const BatchHead &count, size_t head_dim, bool bf16,
                                  unsigned captured) {
    if (count.n_tokens == 0 && !captured) return hipSuccess;
    return head_dim == 64    ? attention<64>(s, a, count, bf16, captured)
           : head_dim == 128 ? attention<128>(s, a, count, bf16, captured)
                             : attention<256>(s, a, count, bf16, captured);
}

}  // namespace th

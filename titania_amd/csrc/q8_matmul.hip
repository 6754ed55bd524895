// Products of 8-bit rows on the matrix cores:
// out[t][r] = x.scale[t] w.scale[r] sum_k x[t][k] w[r][k].
//
// The sums are exact (32-bit integers), so that neither the order nor a split
// of K changes a result; then one conversion to f32 and two products. The
// weights' fragment is the first operand of every product, so that lane l ends
// with weight rows 4 (l / 16) .. + 3 of token l % 16.
//
// Operands are whole fragments (q8.h), 1 KB of consecutive memory each: a wave
// loads one with 16 bytes a lane, into registers or straight into LDS, and
// reads it back from LDS the same way, without bank conflicts and without a
// swizzle. Loads go through a buffer descriptor that ends with the matrix:
// row blocks past its end read as zeros.
#include <algorithm>
#include <iterator>
#include <utility>

#include "device_util.h"
#include "q8.h"

namespace th {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Args {
    const int8_t *w, *x;
    const float *w_scale, *x_scale;
    float *out;
    int n, rows, frags;
    // A split of K (ksplit > 1): part z's sums go to part[z][n][rows].
    int *part;
    int ksplit;
    int keep;  // results stay in the caches (tiles)
};

constexpr unsigned kMostBytes = 0x40000000u;  // a descriptor's range: more than any block's row blocks take
constexpr unsigned kPastEnd = 0xf0000000u;    // an offset past every range: the load gives zero

// The matrix from row block b0 on. (A block of threads reads at most 64 row
// blocks of at most 2 MB.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t blocks_from(const int8_t *p, int rows, int b0, int frags) {
    const size_t block = (size_t)frags * 1024, left = (size_t)((rows + 15) / 16 - b0) * block;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(p) + b0 * block, 0,
                                             (int)(left < kMostBytes ? left : kMostBytes), kBufferRsrcWord3);
}

__device__ __forceinline__ i32x4 load_frag(__amdgpu_buffer_rsrc_t r, unsigned off) {
    return __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}

__device__ __forceinline__ i32x4 mfma(i32x4 w, i32x4 x, i32x4 sum) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, sum, 0, 0, 0);
}

__device__ __forceinline__ f32x4 scaled(i32x4 sum, float xs, float4 ws) {
    return f32x4{(float)sum[0] * xs * ws.x, (float)sum[1] * xs * ws.y, (float)sum[2] * xs * ws.z,
                 (float)sum[3] * xs * ws.w};
}

// Blocks are dealt to the 8 XCDs in turn: a permutation of `count` blocks by
// which each XCD has a range of its own, whose neighbours share its L2.
__device__ __forceinline__ int xcd_range(int lin, int count) {
    const int xcd = lin & 7, q = count >> 3, rest = count & 7;
    return xcd * q + (xcd < rest ? xcd : rest) + (lin >> 3);
}

// Few tokens. A block takes RB row blocks and TB token blocks, its W waves the
// fragments in turn (so that the block reads consecutive memory), U a wave in
// each round of its loop; the waves' sums meet in LDS.
//
// What bounds it is loads in flight: the compiler puts a round's loads between
// its products as registers come free, and each round ends with none. Of a
// round's U (RB + TB) fragments a wave has at first 7 of 10 in flight (one row
// block, one token block), 8 of 15 (one, two), 5 of 20 (two, two) or 6 of 30
// (two, four). One token x 9728 x 2560, captured, takes 3.6 us where the caches
// hold the weights (6.9 TB/s) and 7.1 where 49 such matrices take turns (3.5);
// 151936 x 2560, which no cache holds, 63.5 (6.1); 64 tokens x 2560 x 9728 6.9
// and 13.9. 16 tokens' products take a twentieth of the matrix cores' time in
// which HBM delivers their weights, so that one token is no other case than 16
// (9728 x 2560 from memory 7.1 and 7.7 us). Measured and not kept: K split over
// blocks, the last to arrive adding the parts (64 tokens x 2560 x 9728 back to
// back 9.1 us whole, 9.6 to 14 so).
template <int RB, int TB, int W, int U>
__global__ __launch_bounds__(64 * W) void few_kernel(Args a) {
    __shared__ i32x4 red[W * RB * TB * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (gridDim would add 0.3 us to a launch: an argument block of 256 more bytes.)
    const int tbs = ((a.n + 15) / 16 + TB - 1) / TB, rbs = ((a.rows + 15) / 16 + RB - 1) / RB;
    const int of_xcd = xcd_range(blockIdx.x, rbs * tbs);
    const int rb0 = of_xcd / tbs * RB, tb0 = of_xcd % tbs * TB;
    const unsigned block = (unsigned)a.frags * 1024;
    const __amdgpu_buffer_rsrc_t rw = blocks_from(a.w, a.rows, rb0, a.frags), rx = blocks_from(a.x, a.n, tb0, a.frags);
    unsigned xo[TB];
#pragma unroll
    for (int t = 0; t < TB; ++t) xo[t] = (tb0 + t) * 16 + (lane & 15) < a.n ? t * block + lane * 16 : kPastEnd;
    i32x4 acc[RB][TB] = {};
    for (int f0 = wave; f0 < a.frags; f0 += W * U) {
        i32x4 w[U][RB], x[U][TB];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int f = f0 + u * W;
#pragma unroll
            for (int i = 0; i < RB; ++i)
                w[u][i] = load_frag(rw, f < a.frags ? i * block + f * 1024u + lane * 16 : kPastEnd);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int f = f0 + u * W;
#pragma unroll
            for (int t = 0; t < TB; ++t) x[u][t] = load_frag(rx, f < a.frags ? xo[t] + f * 1024u : kPastEnd);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < RB; ++i)
#pragma unroll
                for (int t = 0; t < TB; ++t) acc[i][t] = mfma(w[u][i], x[u][t], acc[i][t]);
    }
#pragma unroll
    for (int i = 0; i < RB; ++i)
#pragma unroll
        for (int t = 0; t < TB; ++t) red[((wave * RB + i) * TB + t) * 64 + lane] = acc[i][t];
    __syncthreads();
    for (int e = threadIdx.x; e < RB * TB * 64; e += 64 * W) {
        const int q = e >> 6, l = e & 63, t = (tb0 + q % TB) * 16 + (l & 15), r = (rb0 + q / TB) * 16 + (l >> 4) * 4;
        if (t >= a.n || r >= a.rows) continue;
        i32x4 sum = red[e];
#pragma unroll
        for (int k = 1; k < W; ++k) sum += red[k * RB * TB * 64 + e];
        const f32x4 v = scaled(sum, a.x_scale[t], *reinterpret_cast<const float4 *>(a.w_scale + r));
        store4(a.out + (size_t)t * a.rows + r, v, a.rows - r);
    }
}

// The tile of a block: an XCD's tiles go in panels of 8 tiles of tokens, so
// that those that it has in work share operands in its L2.
__device__ __forceinline__ void tile_of_block(int lin, int gr, int gt, int &tr, int &tt) {
    const int i = xcd_range(lin, gr * gt);
    const int high = gt < 8 ? gt : 8, panel = i / (high * gr), in = i % (high * gr);
    const int height = gt - panel * high < high ? gt - panel * high : high;
    tr = in / height;
    tt = panel * high + in % height;
}

// A barrier that does not wait for loads in flight: every wave has waited for
// its own that the others are about to read, and for its reads of what is
// about to be overwritten.
__device__ __forceinline__ void stage_barrier() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// What this wave's lanes have done to LDS comes before what they do next. (The
// hardware keeps a wave's LDS operations in order; this keeps the compiler to it.)
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// Waits until at most VM loads and no LDS reads are outstanding.
template <int VM>
__device__ __forceinline__ void wait_loads_and_lds() {
    static_assert(VM >= 0 && VM < 64, "vmcnt is 6 bits");
    __builtin_amdgcn_s_waitcnt((VM & 15) | (0x7 << 4) | (VM >> 4) << 14);
}

// Many tokens. A block of WM x WN waves takes a tile of BM x BN row blocks
// (weights x tokens), each wave FM x FN of them, K in steps of 128 columns
// (two fragments) through a ring of NS stages in LDS, filled by direct loads
// (1 KB each) that run NS - 1 steps ahead.
//
// A wave goes through a step row by row: FN products with one weight
// fragment, the fragment of kAhead rows on being read meanwhile, and one load
// issued, so that neither LDS nor the memory path sees bursts. The barrier of a
// step comes kAhead rows before its end: by then everything of the stage is in
// registers, its slot is free for new loads, and the first fragments of the
// next stage are read under the last rows' products (1024 tokens x 2560 x
// 9728, us, one row ahead / two / three: 39.6 / 38.9 / 36.8; with all of a
// step's loads and reads at its start, 8192 tokens x 2560 x 9728: 155 -> 149).
//
// Bound by what LDS moves, at the clock that the chip holds under it: a step of
// 160 x 128 takes 1160 cycles, 640 of them with a matrix instruction, whether 61
// CUs work (2.3 GHz, 0.50 us) or 244 (1.85 GHz, 0.62 us), and its 112 KB of
// reads and 36 KB of loads into LDS are 1184 at 128 bytes a cycle. 512 x 9728 x
// 2560 takes 18 us: 20 such steps, the launch (2.4), the first loads, 20 MB of
// results. 8192 tokens x 2560 x 9728 in 320 x 256 tiles back to back 155 us,
// 2630 TOPS, 61% of the cycles with a matrix instruction, 84 MB of results at
// the end. Measured and not kept (before the reads ran three rows ahead): 32 x
// 32 x 32 products (8192 tokens 149 -> 161 us; 6% faster where few CUs work),
// K's halves on two groups of waves (512 x 9728 x 2560 18.5 us), four waves of
// 128 x 128 (410 us).
template <int FM_, int FN_, int WM_, int WN_, int NS_>
struct Tile {
    static constexpr int FM = FM_, FN = FN_, WM = WM_, WN = WN_, NS = NS_, BM = FM * WM, BN = FN * WN;
    static constexpr int kWaves = WM * WN, kFrags = 2 * (BM + BN);                         // of a stage
    static constexpr int kLoads = kFrags / kWaves, kMostLoads = (kFrags + kWaves - 1) / kWaves;  // a wave's
    static constexpr int kRows = 2 * FM, kAhead = FM >= 4 ? 3 : 2;
    static constexpr int kLine = FM * 16 + 4;  // floats of a token in the epilogue, off the banks' period
    static_assert(kMostLoads <= kRows && kWaves * 16 * kLine * 4 <= NS * kFrags * 1024 && NS * kFrags <= 160, "");
    static_assert(kMostLoads >= kAhead, "the prologue issues kAhead loads of the last stage");
};

template <class T>
__global__ __launch_bounds__(64 * T::kWaves) void tile_kernel(Args a, int gr, int gt) {
    constexpr int FM = T::FM, FN = T::FN, NS = T::NS, BM = T::BM, R = T::kRows, D = T::kAhead, L = T::kLoads;
    __shared__ i32x4 ring[NS][T::kFrags][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tr, tt;
    const int z = a.ksplit > 1 ? blockIdx.x / (gr * gt) : 0;
    tile_of_block(blockIdx.x - z * (gr * gt), gr, gt, tr, tt);
    const int all = a.frags / 2, s0 = (int)((long long)all * z / a.ksplit);
    const int rb0 = tr * BM, tb0 = tt * T::BN, steps = (int)((long long)all * (z + 1) / a.ksplit) - s0;
    const unsigned block = (unsigned)a.frags * 1024;
    const __amdgpu_buffer_rsrc_t rw = blocks_from(a.w, a.rows, rb0, a.frags), rx = blocks_from(a.x, a.n, tb0, a.frags);
    // Load j of this wave's for a step: fragment wave + kWaves j of the stage.
    auto load = [&](int step, int slot, int j) {
        const int f = wave + T::kWaves * j, b = f / 2;
        if (j >= L && f >= T::kFrags) return;
        const unsigned col = (unsigned)(2 * (s0 + step) + f % 2) * 1024 + lane * 16;
        auto *to = (__attribute__((address_space(3))) void *)&ring[slot][f][0];
        const bool weights = 2 * BM % T::kWaves == 0 ? j < 2 * BM / T::kWaves : b < BM;
        if (weights) __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, to, 16, (int)(b * block + col), 0, 0, 0);
        else __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, to, 16, (int)((b - BM) * block + col), 0, 0, 0);
    };
    const int wm = wave % T::WM * FM, wn = wave / T::WM * FN;  // this wave's first row block and token block
    auto read_w = [&](int slot, int r) { return ring[slot][(wm + r % FM) * 2 + r / FM][lane]; };
    auto read_x = [&](int slot, int k, int j) { return ring[slot][(BM + wn + j) * 2 + k][lane]; };

    i32x4 acc[FM][FN] = {};
#pragma unroll
    for (int s = 0; s < NS - 1; ++s)
        if (s < steps) {
#pragma unroll
            for (int j = 0; j < T::kMostLoads; ++j) load(s, s, j);
        }
    if (NS - 1 < steps) {
#pragma unroll
        for (int j = 0; j < D; ++j) load(NS - 1, NS - 1, j);
        wait_loads_and_lds<(NS - 2) * L + (D < L ? D : L)>();
    } else {
        wait_loads_and_lds<0>();
    }
    stage_barrier();
    i32x4 x[2][FN], w[R], next[D];
#pragma unroll
    for (int j = 0; j < FN; ++j) x[0][j] = read_x(0, 0, j);
#pragma unroll
    for (int r = 0; r < D; ++r) w[r] = read_w(0, r);
    int cur = 0;
    for (int step = 0; step < steps; ++step) {
        const int nxt = cur + 1 == NS ? 0 : cur + 1, prv = cur == 0 ? NS - 1 : cur - 1;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int k = r / FM, i = r % FM;
            if (r == R - D) {
                if (step + NS - 1 < steps) wait_loads_and_lds<(NS - 2) * L>();
                else wait_loads_and_lds<0>();
                stage_barrier();
#pragma unroll
                for (int j = 0; j < FN; ++j) x[0][j] = read_x(nxt, 0, j);
            }
            if (r == 0) {
#pragma unroll
                for (int j = 0; j < FN; ++j) x[1][j] = read_x(cur, 1, j);
            }
            if (r + D < R) w[r + D] = read_w(cur, r + D);
            else next[r + D - R] = read_w(nxt, r + D - R);
            // The loads of step + NS go where this step was, from its barrier on.
            if (r >= R - D) {
                if (step + NS < steps) load(step + NS, cur, r - (R - D));
            } else if (r + D < T::kMostLoads) {
                if (step - 1 + NS < steps) load(step - 1 + NS, prv, r + D);
            }
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = mfma(w[r], x[k][j], acc[i][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int r = 0; r < D; ++r) w[r] = next[r];
        cur = nxt;
    }

    // 16 tokens at a time through LDS, so that a token's FM * 16 values are
    // stored side by side: whole lines, where a lane's own four would be a
    // part of one (a 256 x 256 tile's stores took 10 us, now 5).
    const int lt = lane & 15, lr = lane >> 4 << 2, r0 = (rb0 + wm) * 16, t0 = (tb0 + wn) * 16;
    const int last = (a.rows + 15) / 16 * 16 - 4;
    float4 ws[FM];
    float xs[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) ws[i] = *reinterpret_cast<const float4 *>(a.w_scale + min(r0 + i * 16 + lr, last));
#pragma unroll
    for (int j = 0; j < FN; ++j) xs[j] = a.x_scale[min(t0 + j * 16 + lt, a.n - 1)];
    __syncthreads();
    float *lines = reinterpret_cast<float *>(ring) + wave * 16 * T::kLine;
    float *out = a.ksplit > 1 ? reinterpret_cast<float *>(a.part + (size_t)z * a.n * a.rows) : a.out;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        if (j) wave_lds_order();  // the lines have been read
#pragma unroll
        for (int i = 0; i < FM; ++i)
            *reinterpret_cast<f32x4 *>(lines + lt * T::kLine + i * 16 + lr) =
                a.ksplit > 1 ? __builtin_bit_cast(f32x4, acc[i][j]) : scaled(acc[i][j], xs[j], ws[i]);
        wave_lds_order();  // other lanes read them
#pragma unroll
        for (int q = 0; q < FM; ++q) {
            const int e = q * 64 + lane, t = e / (FM * 4), c = e % (FM * 4) * 4;
            const f32x4 v = *reinterpret_cast<const f32x4 *>(lines + t * T::kLine + c);
            if (t0 + j * 16 + t >= a.n || r0 + c >= a.rows) continue;
            float *o = out + (size_t)(t0 + j * 16 + t) * a.rows + r0 + c;
            if (a.keep) store4(o, v, a.rows - r0 - c);
            else store4<true>(o, v, a.rows - r0 - c);
        }
    }
}

// The sums of a split of K, four rows of a token a thread (rows % 4 == 0) or
// one. (1024 tokens x 1024 x 9728, 64 tiles of 128 x 128: 35.8 us whole, 22.7
// in four parts with this.)
template <int V>
__global__ __launch_bounds__(256) void join_kernel(Args a) {
    const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * V, m = (size_t)a.n * a.rows;
    if (i >= m) return;
    const int t = (int)(i / a.rows), r = (int)(i % a.rows);
    if constexpr (V == 4) {
        i32x4 sum = {};
        for (int z = 0; z < a.ksplit; ++z) sum += *reinterpret_cast<const i32x4 *>(a.part + z * m + i);
        *reinterpret_cast<f32x4 *>(a.out + i) =
            scaled(sum, a.x_scale[t], *reinterpret_cast<const float4 *>(a.w_scale + r));
    } else {
        int sum = 0;
        for (int z = 0; z < a.ksplit; ++z) sum += a.part[z * m + i];
        a.out[i] = (float)sum * a.x_scale[t] * a.w_scale[r];
    }
}

unsigned ceil_div(unsigned a, unsigned b) { return (a + b - 1) / b; }
unsigned blocks_of(int rows, unsigned each) { return ceil_div(ceil_div((unsigned)rows, 16), each); }

template <int RB, int TB, int W>
void few(hipStream_t s, const Args &a) {
    few_kernel<RB, TB, W, 5><<<blocks_of(a.rows, RB) * blocks_of(a.n, TB), 64 * W, 0, s>>>(a);
}

template <class T>
void tiles(hipStream_t s, const Args &a) {
    const int gr = (int)blocks_of(a.rows, T::BM), gt = (int)blocks_of(a.n, T::BN);
    tile_kernel<T><<<(unsigned)gr * (unsigned)gt * (unsigned)a.ksplit, 64 * T::kWaves, 0, s>>>(a, gr, gt);
    if (a.ksplit == 1) return;
    const size_t m = (size_t)a.n * a.rows;
    if (a.rows % 4 == 0) join_kernel<4><<<(unsigned)((m / 4 + 255) / 256), 256, 0, s>>>(a);
    else join_kernel<1><<<(unsigned)((m + 255) / 256), 256, 0, s>>>(a);
}

// About how long a launch takes, in us, from its shape alone. The constants
// are fitted to back-to-back launches of every variant. Over 17 matrices (7 x
// 3000 to 16384 x 2048) and up to 15 counts of tokens (20 to 8192), 254 products,
// the variant that they choose takes 1.02 times the fastest one's time in the
// geometric mean and 1.64 times at most (2048 tokens x 51 x 6076 9.6 us for 5.9;
// 1500 x 300 x 16000 30.7 for 21.0, 1024 x 1024 x 9728 25.3 for 18.3, all others
// within 1.31).
constexpr double kLaunch = 2.4;
constexpr unsigned kCus = 256;

// The work of the CUs and the matrices' way to and from them, which mostly overlap.
double overlapped(double work, double bytes) {
    const double way = bytes / 9.0e6;
    return kLaunch + std::max(work, way) + 0.15 * std::min(work, way);
}

// What the estimates look at.
struct Shape {
    unsigned rows, tokens, steps;       // row blocks of the weights and of the tokens, steps of 128 columns
    double results;                     // values
    double weights_and_results, token_bytes;
    explicit Shape(const Args &a)
        : rows(blocks_of(a.rows, 1)), tokens(blocks_of(a.n, 1)), steps(a.frags / 2), results((double)a.n * a.rows),
          weights_and_results(1024.0 * rows * a.frags + 4 * results), token_bytes(1024.0 * tokens * a.frags) {}
    size_t tiles(unsigned bm, unsigned bn) const { return (size_t)ceil_div(rows, bm) * ceil_div(tokens, bn); }
};

// Few tokens: what a CU takes in through its memory path, block after block;
// each group of row blocks reads the tokens again, mostly from L2.
double few_us(const Shape &a, int rb, int tb) {
    const size_t count = a.tiles(rb, tb);
    const double groups = ceil_div(a.rows, rb), rounds = (double)count / kCus;
    const double work = a.steps * (rb + tb) / 42.0 + 0.75 + 0.04 * rb * tb;
    return overlapped((0.73 * ((count + kCus - 1) / kCus) + 0.27 * std::max(rounds, 1.0)) * work,
                      a.weights_and_results + a.token_bytes * (1 + 0.11 * (groups - 1)));
}

struct TileVariant {
    int bm, bn, products;  // row blocks, token blocks, products of a wave for 64 columns
    int resident;          // tiles that a CU holds at once
    void (*launch)(hipStream_t, const Args &);
};
template <int FM, int FN, int WM, int WN, int NS>
constexpr TileVariant variant() {
    using T = Tile<FM, FN, WM, WN, NS>;
    return {T::BM, T::BN, FM * FN, T::kFrags * NS <= 80 ? 2 : 1, tiles<T>};
}
// Heights in small steps: as a CU holds one block, a launch takes whole rounds
// of 256 tiles, and the height that leaves the least of the last round idle
// wins (8192 tokens x 2560 x 9728: 320 x 256 tiles, one round, 148 us; 256 x
// 256, 1.25 rounds, 204 us; 224 x 256, 1.5 rounds, 188 us).
constexpr TileVariant kTiles[] = {
    variant<2, 1, 4, 2, 4>(), variant<2, 2, 4, 2, 4>(), variant<4, 2, 2, 4, 2>(), variant<4, 2, 2, 4, 4>(),
    variant<5, 2, 2, 4, 4>(), variant<6, 2, 2, 4, 3>(), variant<5, 4, 2, 4, 3>(),
    variant<6, 4, 2, 4, 2>(), variant<7, 4, 2, 4, 2>(), variant<8, 4, 2, 4, 2>(), variant<10, 4, 2, 4, 2>(),
};

// Tiles: rounds of a tile a CU, each with its steps of K and its epilogue (the
// variant of which a CU holds two: a round of both takes 1.29 times one tile's
// time; with one it waits for its short ring). A split's sums go out and come
// in again.
inline double tile_us(const Shape &a, const TileVariant &v, size_t tiles, unsigned ksplit) {
    const size_t count = tiles * ksplit, at_once = (size_t)kCus * v.resident;
    const double steps = ceil_div(a.steps, ksplit), rounds = (count + at_once - 1) / at_once;
    const double one = steps * (0.306 + 0.029 * v.products) + 0.6 + 0.15 * v.products;
    const double us = overlapped(rounds * one * (v.resident == 1 ? 1.0 : count > kCus ? 1.29 : 1.08),
                                 a.weights_and_results + a.token_bytes);
    return ksplit == 1 ? us : us + 3.8 + ksplit * 8.0 * a.results / 3.9e6;
}

struct FewVariant {
    int rb, tb;
    void (*launch)(hipStream_t, const Args &);
};
// More waves where a block has much to read and the chip is not full, fewer
// where there is little (one token, us with 4 / 8 / 16 waves: 1024 x 1024 2.4 /
// 2.6 / 3.2, 2560 x 9728 7.2 / 6.1 / 5.7).
constexpr FewVariant kFew[] = {
    {1, 1, few<1, 1, 8>}, {1, 2, few<1, 2, 8>}, {2, 2, few<2, 2, 8>}, {2, 4, few<2, 4, 8>},  // as the estimate says
    {1, 1, few<1, 1, 4>}, {1, 2, few<1, 2, 4>},                                              // for short rows
    {1, 1, few<1, 1, 16>},                                                                   // for long ones
};

// What a product takes: a variant of kFew, or of kTiles with K in ksplit parts.
struct Choice {
    const FewVariant *few;
    const TileVariant *tile;
    int ksplit;
};

// One instance a variant, so that their sizes are constants: the whole choice
// takes a call about 75 ns, with a loop over the variants 210.
template <size_t I>
inline void consider_tile(const Shape &a, size_t part_len, Choice &best, double &least) {
    constexpr TileVariant v = kTiles[I];
    const size_t tiles = a.tiles(v.bm, v.bn);
    if (const double us = tile_us(a, v, tiles, 1); us < least) least = us, best = {nullptr, &kTiles[I], 1};
    // As many parts as fill the chip, of two steps at least.
    if (tiles > kCus / 2) return;
    const unsigned z = std::min({kCus / (unsigned)tiles, a.steps / 2, 16u});
    if (z < 2 || z * a.results > (double)part_len) return;
    if (const double us = tile_us(a, v, tiles, z); us < least) least = us, best = {nullptr, &kTiles[I], (int)z};
}
template <size_t... I>
void consider_tiles(const Shape &a, size_t part_len, Choice &best, double &least, std::index_sequence<I...>) {
    (consider_tile<I>(a, part_len, best, least), ...);
}

Choice choose(const Args &args, size_t part_len) {
    const bool is_short = args.frags <= 24;
    if (args.n <= 16) {
        const bool is_long = args.frags >= 128 && blocks_of(args.rows, 1) <= kCus;
        return {&kFew[is_short ? 4 : is_long ? 6 : 0], nullptr, 1};
    }
    const Shape a(args);
    Choice best{};
    double least = 1e30;
    for (int i = 0; i < 4; ++i)
        if (const double us = few_us(a, kFew[i].rb, kFew[i].tb); us < least)
            least = us, best = {&kFew[is_short && i < 2 ? i + 4 : i], nullptr, 1};
    consider_tiles(a, part_len, best, least, std::make_index_sequence<std::size(kTiles)>());
    return best;
}

// Results that a tile stores in the caches' normal order: those that the L2s do
// not hold (which would write them back all at once at the kernel's end), and
// of which two and their operands find room in the 256 MB of the memory-side
// cache until they are read. (Three gated MLPs of 2560 columns in turn, us each
// so / with nontemporal stores. 9728 between, results of 23.8 MB 94.6 / 93.4,
// 31.5 119.5 / 121.8, 33.4 120.7 / 122.9, 38.0 128.0 / 131.4, 48.2 151.8 /
// 154.5, 55.7 161.6 / 167.9, 63.1 182.3 / 187.0, 66.8 192.2 / 192.3, 76.0 206.6 /
// 204.3; 4096 between, 28.1 101.5 / 100.9, 32.0 107.7 / 111.8, 46.9 147.2 /
// 153.4, 62.5 175.3 / 180.6, 65.6 194.1 / 193.5, 78.1 239.0 / 235.5.)
constexpr size_t kKeepFrom = (size_t)32 << 20, kKeepTo = (size_t)64 << 20;

}  // namespace

int matmul_q8_variant(size_t n, size_t rows, size_t cols, size_t part_len, int *ksplit) {
    Args a{};
    a.n = (int)n, a.rows = (int)rows, a.frags = (int)q8_frags(cols);
    const Choice c = choose(a, part_len);
    *ksplit = c.ksplit;
    return c.few ? (int)(c.few - kFew) : (int)(std::size(kFew) + (c.tile - kTiles));
}

hipError_t launch_matmul_q8(hipStream_t s, float *out, const th_q8 &w, const th_q8 &x, int *part, size_t part_len) {
    if (x.rows == 0 || w.rows == 0) return hipSuccess;
    Args a{w.ptr, x.ptr, w.scale, x.scale, out, (int)x.rows, (int)w.rows, (int)q8_frags(w.cols), part, 1, 0};
    const Choice c = choose(a, part_len);
    a.ksplit = c.ksplit;
    const size_t bytes = x.rows * w.rows * sizeof(float);
    a.keep = c.ksplit == 1 && bytes >= kKeepFrom && bytes <= kKeepTo;
    (c.tile ? c.tile->launch : c.few->launch)(s, a);
    return hipGetLastError();
}

}  // namespace th

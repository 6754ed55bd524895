// Rows in 8 bits: f32 rows, bf16 weights, rmsnorm(x + y) and silu(gate) * up
// as integers with a scale a row, and the values that such rows stand for.
//
// Of a row v with A = max |v|, the integers are those nearest to 127 v / A
// (ties to even) and the scale is A / 127 in f32; where that rounds to zero, so
// do the integers. The quotients are decided in 64 bits, so that the integers
// are the definition's whatever the launch. For rmsnorm, v_c = r x_c g_c with
// one positive r a row, which the quotients lose: 127 x_c g_c / max |x g|, whose
// products are exact in 64 bits.
#include <algorithm>
#include <cfloat>

#include "device_util.h"
#include "q8.h"

namespace th {
namespace {

// The nearest integer to 127 v / most. inv: 127 / most. v * inv is off by at
// most 127 * 2^-52, so only what lies within 1e-12 of a border is divided.
__device__ __forceinline__ int nearest(double v, double most, double inv) {
    double t = v * inv;
    if (fabs(fabs(t - trunc(t)) - 0.5) < 1e-12) t = v * 127.0 / most;
    return (int)rint(t);
}

// Four values from column c of a row, which starts at any multiple of 4 bytes,
// zeros past its end. NT: past the caches' normal order.
template <bool NT>
__device__ __forceinline__ void load4(const float *row, int c, int cols, float (&v)[4]);

// What a row is made of. value: the 64-bit value (of the norm without its
// factor r) at flat index i, column c. load: a thread's f32 values, N times four
// columns from column c0 + 4 threadIdx.x on; kOff is how far they may be off,
// relative to the value; a and b have what value64 makes the 64-bit value of.
template <bool NT>
struct RowsSource {
    static constexpr bool kNorm = false, kNt = NT;
    static constexpr float kOff = 0;
    const float *x;
    static __device__ double value64(float a, float) { return (double)a; }
    __device__ double value(size_t i, size_t) const { return (double)x[i]; }
    template <int N, int T>
    __device__ void load(size_t row, int c0, int cols, float (&v)[N][4], float (&a)[N][4], float (&)[N][4], double &,
                         int &) const {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            load4<NT>(x + row * cols, c0 + 4 * (threadIdx.x + T * k), cols, v[k]);
#pragma unroll
            for (int j = 0; j < 4; ++j) a[k][j] = v[k][j];
        }
    }
};

struct WeightSource {
    static constexpr bool kNorm = false;
    const uint16_t *w;
    __device__ double value(size_t i, size_t) const { return (double)bf16_to_f32(w[i]); }
};

template <bool NT>
struct NormSource {
    static constexpr bool kNorm = true, kNt = NT;
    static constexpr float kOff = 1.0f / (1 << 24);
    float *x;
    const float *y;
    const uint16_t *g;
    float eps;
    static __device__ double value64(float a, float b) { return (double)a * (double)b; }
    __device__ double value(size_t i, size_t c) const { return value64(x[i], bf16_to_f32(g[c])); }
    template <int N, int T>
    __device__ void load(size_t row, int c0, int cols, float (&v)[N][4], float (&a)[N][4], float (&b)[N][4],
                         double &sum, int &odd) const;
};

template <bool NT>
struct SiluSource {
    static constexpr bool kNorm = false, kNt = NT;
    // The exponential and the reciprocal within 2^-23, the exponential's
    // correction, its product, the sum and the two products within 2^-24: 4.5
    // 2^-23 and a little for their products. (silu alone, over every f32 gate
    // from -80 up: 2.13 2^-23 at most, where this allows 4.)
    static constexpr float kOff = 5.0f / (1 << 23);
    const float *gate, *up;
    static __device__ double value64(float a, float b) {
        const double g = (double)a;
        return g / (1.0 + exp(-g)) * (double)b;
    }
    __device__ double value(size_t i, size_t) const { return value64(gate[i], up[i]); }
    template <int N, int T>
    __device__ void load(size_t row, int c0, int cols, float (&v)[N][4], float (&a)[N][4], float (&b)[N][4], double &,
                         int &odd) const {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            load4<NT>(gate + row * cols, c0 + 4 * (threadIdx.x + T * k), cols, a[k]);
            load4<NT>(up + row * cols, c0 + 4 * (threadIdx.x + T * k), cols, b[k]);
        }
        float least = 0, most_up = 0;
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // exp(-g) = 2^t (1 + d ln 2): t = -g / ln 2 rounded, d what that
                // left and what the f32 of 1 / ln 2 lacks.
                const float g = a[k][j], t = g * -1.44269502f;
                const float d = fmaf(g, -1.92596303e-8f, fmaf(g, -1.44269502f, -t));
                const float e = __builtin_amdgcn_exp2f(t);
                v[k][j] = g * __builtin_amdgcn_rcpf(1.f + fmaf(e, d * 0.693147182f, e)) * b[k][j];
                least = fminf(least, g);
                most_up = fmaxf(most_up, fabsf(b[k][j]));
            }
        // exp(-g) past f32; or silu(g) below its normal numbers, off by 2^-150,
        // times what makes that more than 2^-26 of the least maximum taken.
        odd |= least < -80.f || most_up > 0x1p24f;
    }
};

// Block b's row. Blocks are dealt to the 8 XCDs in turn; with 128 rows or more,
// an XCD takes 16 consecutive rows at a time, so that the pieces of 16 bytes
// that each row has of a fragment's lines meet in one L2.
__device__ __forceinline__ size_t row_of_block(unsigned b, bool grouped) {
    return grouped ? ((size_t)(b >> 7) * 8 + (b & 7)) * 16 + (b >> 3 & 15) : b;
}

// Maxima and sums over a block of W waves, the same in every thread.
template <int W>
struct Reduced {
    double most[W], sum[W];
    int flag[W];
};
template <int W>
__device__ __forceinline__ void reduce(Reduced<W> &sh, double &most, double &sum, int &flag) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        most = fmax(most, __shfl_xor(most, o, 64));
        sum += __shfl_xor(sum, o, 64);
    }
    flag = __any(flag);
    if ((threadIdx.x & 63) == 0) {
        sh.most[threadIdx.x >> 6] = most;
        sh.sum[threadIdx.x >> 6] = sum;
        sh.flag[threadIdx.x >> 6] = flag;
    }
    __syncthreads();
    most = sum = 0;
    flag = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        most = fmax(most, sh.most[w]);
        sum += sh.sum[w];
        flag |= sh.flag[w];
    }
}

// The scale of a row whose largest value is most (the norm's: times r), or NaN,
// with bad set, where the row is to be marked.
template <class Source>
__device__ __forceinline__ float scale_of(const Source &src, double most, double sum, int cols, int &bad) {
    double top = most;
    if constexpr (Source::kNorm) top = most == 0 ? 0 : most / sqrt(sum / cols + (double)src.eps);
    const float s = (float)(top / 127.0);
    bad |= !(s <= FLT_MAX);
    return bad ? __builtin_nanf("") : s;
}

// A row in 64 bits, read once for its maximum and again for its integers: any
// row, by W waves. add: y is to be added first.
template <class Source, int W>
__device__ __forceinline__ void any_row(const Source &src, size_t row, int8_t *__restrict__ q,
                                        float *__restrict__ scale, int cols, int frags, bool add) {
    __shared__ Reduced<W> sh;
    double most = 0, sum = 0;
    int bad = 0;
    for (int c = threadIdx.x; c < cols; c += 64 * W) {
        const size_t i = row * cols + c;
        if constexpr (Source::kNorm) {
            float v = src.x[i];
            if (add && src.y) src.x[i] = v += src.y[i];
            sum += (double)v * (double)v;
        }
        const double v = fabs(src.value(i, c));
        bad |= !(v <= DBL_MAX);
        most = fmax(most, v);
    }
    reduce(sh, most, sum, bad);
    const float s = scale_of(src, most, sum, cols, bad);
    if (threadIdx.x == 0) scale[row] = s;
    const double inv = 127.0 / most;
    for (int c = threadIdx.x; c < cols; c += 64 * W) {
        const int v = bad || s == 0 ? 0 : nearest(src.value(row * cols + c, c), most, inv);
        q[q8_at(row, c, frags)] = (int8_t)v;
    }
}

// Rows longer than registers hold, and weights (once a weight's life).
template <class Source, int W>
__global__ __launch_bounds__(64 * W) void any_row_kernel(Source src, int8_t *__restrict__ q, float *__restrict__ scale,
                                                         size_t row0, int cols, int frags) {
    any_row<Source, W>(src, row0 + blockIdx.x, q, scale, cols, frags, true);
}

template <bool NT>
__device__ __forceinline__ void load4(const float *row, int c, int cols, float (&v)[4]) {
    if (c + 4 <= cols) {
        const auto *at = reinterpret_cast<const f32x4_any *>(row + c);
        const f32x4_any l = NT ? __builtin_nontemporal_load(at) : *at;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = l[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = c + j < cols ? row[c + j] : 0.f;
    }
}

template <bool NT>
template <int N, int T>
__device__ void NormSource<NT>::load(size_t row, int c0, int cols, float (&v)[N][4], float (&a)[N][4], float (&b)[N][4],
                                 double &sum, int &odd) const {
    float u[N][4];
    alignas(8) uint16_t gain[N][4];
    float *xr = x + row * cols;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int c = c0 + 4 * (threadIdx.x + T * k);
        load4<NT>(xr, c, cols, a[k]);
        if (y) load4<NT>(y + row * cols, c, cols, u[k]);
        if (c + 4 <= cols) {
            *reinterpret_cast<uint2 *>(gain[k]) = *reinterpret_cast<const uint2 *>(g + c);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) gain[k][j] = c + j < cols ? g[c + j] : 0;
        }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int c = c0 + 4 * (threadIdx.x + T * k);
        if (y) {
#pragma unroll
            for (int j = 0; j < 4; ++j) a[k][j] += u[k][j];
            store4(xr + c, f32x4_any{a[k][0], a[k][1], a[k][2], a[k][3]}, cols - c);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double d = (double)a[k][j];
            b[k][j] = bf16_to_f32(gain[k][j]);
            sum = fma(d, d, sum);
            v[k][j] = a[k][j] * b[k][j];
        }
    }
}

// x[i / 4][i % 4], of registers (by masks, which no compiler turns into an
// array in memory).
template <int N>
__device__ __forceinline__ float pick(const float (&x)[N][4], int i) {
    unsigned r = 0;
#pragma unroll
    for (int e = 0; e < 4 * N; ++e) r |= __float_as_uint(x[e / 4][e % 4]) & (unsigned)-(int)(i == e);
    return __uint_as_float(r);
}

// A barrier for what is in LDS: it waits for no store to memory.
__device__ __forceinline__ void lds_barrier() {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt 0
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// A wave's sum in 64 bits, left in lane 63: wave_sum_dpp's steps.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ double dpp_add_f64(double v) {
    const long long b = __double_as_longlong(v);
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, ROW_MASK, 0xf, false);
    const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROW_MASK, 0xf, false);
    return v + __longlong_as_double((long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_f64(double v) {
    v = dpp_add_f64<0xB1, 0xf>(v);
    v = dpp_add_f64<0x4E, 0xf>(v);
    v = dpp_add_f64<0x124, 0xf>(v);
    v = dpp_add_f64<0x128, 0xf>(v);
    v = dpp_add_f64<0x142, 0xa>(v);
    return dpp_add_f64<0x143, 0xc>(v);
}

// Rows of up to 256 W N G columns, one block of W waves a row, in G parts of N
// times four columns a thread, whose values are held in registers, so that the
// row is read once. Of a row in one part so is what they are formed from; of
// one in several that is read again for the few values that need it.
//
// Bound by memory (norm 8192 x 2560 48.4 us, 5.6 TB/s; rows 8192 x 4096 30.9,
// 5.4; silu 2048 x 9728 37.8, 4.7); one row by its chain of loads, maxima and
// barriers on one CU (norm of 2560 3.4 us, silu of 9728 5.5). What 64 bits
// decide is found in 32 first: a value's f32 is off by at most Source::kOff of
// it, and the quotient by 127 times that and three roundings (the largest
// value's, the factor's, the product's), so only values within twice kOff of
// the largest are compared in 64 bits, and only quotients within 127 kNear of
// a border are formed again (2 in 10000 for silu). With 64 bits
// throughout and a second pass over memory the same took 90, 88 and 85 us.
// Rows on which f32 does not hold what 64 bits do (values past 1e38 or not
// finite, none as large as 1e-30, arguments at which silu leaves f32) are taken
// by any_row.
template <class Source, int W, int N, int G>
__global__ __launch_bounds__(64 * W, G > 5 ? 4 : 1) void rows_kernel(Source src, int8_t *__restrict__ q, float *__restrict__ scale,
                                                      size_t row0, size_t rows, int cols, int frags,
                                                      bool grouped) {
    constexpr int T = 64 * W, M = N * G;
    constexpr float kNear = Source::kOff + 5.0f / (1 << 24);
    __shared__ alignas(16) float red_max[W];
    __shared__ alignas(16) double red_sum[W];
    __shared__ alignas(16) unsigned long long red_exact[W];
    const size_t row = row0 + row_of_block(blockIdx.x, grouped);
    if (row >= rows) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float v[M][4], a[N][4], b[N][4];
    double sum = 0;
    int odd = 0;
    if constexpr (G == 1) {
        src.template load<N, T>(row, 0, cols, v, a, b, sum, odd);
    } else {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            float(&part)[N][4] = *reinterpret_cast<float(*)[N][4]>(v[g * N]);
            src.template load<N, T>(row, 4 * T * N * g, cols, part, a, b, sum, odd);
            __builtin_amdgcn_sched_barrier(0);  // a part's inputs are gone before the next one's come
        }
    }
    auto column = [](int i) { return 4 * (int)(threadIdx.x + T * (i >> 2)) + (i & 3); };
    auto value64 = [&](int i) {
        if constexpr (G == 1) return Source::value64(pick(a, i), pick(b, i));
        else return src.value(row * cols + column(i), column(i));
    };
    float m = 0, none = 0;  // 0 * v: NaN where v is not finite
#pragma unroll
    for (int k = 0; k < M; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            none = fmaf(v[k][j], 0.f, none);
            m = fmaxf(m, fabsf(v[k][j]));
        }
    const float own = odd || none != 0 || m >= 1e38f ? INFINITY : m;
    m = wave_max_dpp(own);
    if constexpr (Source::kNorm) sum = wave_sum_f64(sum);
    if (lane == 63) {
        red_max[wave] = m;
        if constexpr (Source::kNorm) red_sum[wave] = sum;
    }
    if (lane == 0) red_exact[wave] = 0;
    lds_barrier();
    sum = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        m = fmaxf(m, red_max[w]);
        if constexpr (Source::kNorm) sum += red_sum[w];
    }
    if (!(m < INFINITY && m >= 1e-30f)) {
        __syncthreads();  // x, which other threads wrote
        any_row<Source, W>(src, row, q, scale, cols, frags, false);
        return;
    }
    double most = m;
    if constexpr (Source::kOff > 0) {
        // The largest in 64 bits: nearly always one thread has a candidate, one.
        // Positive doubles are ordered as their bits are.
        const float reach = m * (1 - 2 * Source::kOff - 1.0f / (1 << 23));
        if (own >= reach) {
            uint64_t near = 0;
#pragma unroll
            for (int i = 0; i < 4 * M; ++i) near |= (uint64_t)(fabsf(v[i / 4][i % 4]) >= reach) << i;
            for (; near; near &= near - 1) {
                const double d = fabs(value64(__builtin_ctzll(near)));
                atomicMax(&red_exact[wave], (unsigned long long)__double_as_longlong(d));
            }
        }
        lds_barrier();
        unsigned long long bits = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) bits = max_u64(bits, red_exact[w]);
        most = __longlong_as_double((long long)bits);
    }
    const float inv32 = 127.0f / (float)most;
    char4 *out = reinterpret_cast<char4 *>(q);
    constexpr float kBorder = 0.5f - 127 * kNear;
    float furthest = 0;
#pragma unroll
    for (int k = 0; k < M; ++k) {
        const int c = 4 * (threadIdx.x + T * k);
        if (c >= cols) break;
        int n[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float t = v[k][j] * inv32, r = rintf(t);
            n[j] = (int)r;
            furthest = fmaxf(furthest, fabsf(t - r));
        }
        out[q8_at(row, c, frags) / 4] = make_char4((char)n[0], (char)n[1], (char)n[2], (char)n[3]);
    }
    if (furthest > kBorder) {
        uint64_t near = 0;
#pragma unroll
        for (int i = 0; i < 4 * M; ++i) {
            const float t = v[i / 4][i % 4] * inv32;
            near |= (uint64_t)(fabsf(t - rintf(t)) > kBorder && column(i) < cols) << i;
        }
        const double inv = 127.0 / most;
        for (; near; near &= near - 1) {
            const int i = __builtin_ctzll(near);
            q[q8_at(row, column(i), frags)] = (int8_t)nearest(value64(i), most, inv);
        }
    }
    int bad = 0;
    const float s = scale_of(src, most, sum, cols, bad);
    if (threadIdx.x == 0) scale[row] = s;
    if (bad || s == 0)
        for (int c = 4 * threadIdx.x; c < cols; c += 4 * T) out[q8_at(row, c, frags) / 4] = make_char4(0, 0, 0, 0);
}

// A block a 16 rows x 256 columns: four rows of four columns a thread. Stores
// of 16 bytes past the caches' normal order (8192 x 4096 24.5 us; 46.7 with the
// row ends' 4 and 8 bytes throughout, which the compiler makes of a packed
// struct).
__global__ __launch_bounds__(256) void dequantize_kernel(float *__restrict__ out, const int8_t *__restrict__ q,
                                                         const float *__restrict__ scale, size_t rows, int cols,
                                                         int frags, int parts) {
    const size_t row0 = (size_t)(blockIdx.x / parts) * 16 + (threadIdx.x >> 6) * 4;
    const int c = ((int)(blockIdx.x % parts) * 64 + (threadIdx.x & 63)) * 4;
    if (c >= cols || row0 >= rows) return;
    char4 v[4];
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const size_t row = row0 + i < rows ? row0 + i : rows - 1;
        v[i] = *reinterpret_cast<const char4 *>(q + q8_at(row, c, frags));
        s[i] = scale[row];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (row0 + i >= rows) return;
        float *o = out + (row0 + i) * cols + c;
        store4<true>(o, f32x4_any{v[i].x * s[i], v[i].y * s[i], v[i].z * s[i], v[i].w * s[i]}, cols - c);
    }
}

struct __attribute__((packed, aligned(1))) Loose16 {
    uint32_t w[4];
};

// Row-major integers to the fragments' order (IN) or back, 16 columns a thread.
template <bool IN>
__global__ __launch_bounds__(256) void reorder_kernel(int8_t *__restrict__ q, int8_t *__restrict__ plain, size_t row0,
                                                      size_t rows, int cols, int frags) {
    const int pieces = (cols + 15) / 16;
    const size_t e = (size_t)blockIdx.x * 256 + threadIdx.x, r = e / pieces;
    if (r >= rows) return;
    const int c = (int)(e % pieces) * 16;
    int8_t *in = plain + r * cols + c, *at = q + q8_at(row0 + r, c, frags);
    if (c + 16 <= cols) {
        if (IN) *reinterpret_cast<Loose16 *>(at) = *reinterpret_cast<const Loose16 *>(in);
        else *reinterpret_cast<Loose16 *>(in) = *reinterpret_cast<const Loose16 *>(at);
    } else {
        for (int j = 0; c + j < cols; ++j) (IN ? at : in)[j] = (IN ? in : at)[j];
    }
}

// Inputs of half the 256 MB of the memory-side cache are read past the caches'
// normal order (norm 8192 x 2560 from memory 53 -> 48 us; a gated MLP of 8192
// tokens x 2560 x 9728 733 -> 695, of 4096 388 -> 376, of 2048 208 -> 205);
// smaller ones not: they may still be there (84 MB quantized again and again
// 16.7 us, 20.7 so read). At the limit (us in the normal order / past it): from
// memory norm of 98 MB 34.7 / 32.4, 117 40.1 / 37.3, 128 42.9 / 40.3, silu of
// 128 33.8 / 33.1; again and again, norm 28.3 / 32.4, 32.8 / 37.3, 35.4 / 40.2,
// silu 28.9 / 31.5; three MLPs in turn, of which the silu reads 111 MB 162.7 /
// 162.5, 126 182.3 / 183.4, 134 195.2 / 191.9, 152 207.6 / 204.8. Rows alone
// gain nothing by it (129 MB 31.9 / 33.2 from memory, 24.6 / 32.6 again).
constexpr size_t kPastCaches = (size_t)128 << 20;

// Rows a launch of up to 1024 threads a row, and blocks of one of 256 threads a
// block: fewer than 2^32 threads. (2^25 rows of 1793 values, which 288 GB hold,
// would be 2^24 of those blocks.)
constexpr size_t kRowsALaunch = (size_t)1 << 21, kBlocksALaunch = (size_t)1 << 22;
static_assert(kRowsALaunch * 1024 < (size_t)1 << 32 && kBlocksALaunch * 256 < (size_t)1 << 32, "");

template <class Source, int W, int N, int G = 1>
void launch_held(hipStream_t s, const th_q8 &q, const Source &src) {
    for (size_t r = 0; r < q.rows; r += kRowsALaunch) {
        const size_t rows = std::min(q.rows - r, kRowsALaunch);
        const bool grouped = rows >= 128;
        const size_t blocks = grouped ? (rows + 127) / 128 * 128 : rows;
        rows_kernel<Source, W, N, G><<<(unsigned)blocks, 64 * W, 0, s>>>(src, q.ptr, q.scale, r, q.rows, (int)q.cols,
                                                                         (int)q8_frags(q.cols), grouped);
    }
}

template <class Source, int W>
void launch_any(hipStream_t s, const th_q8 &q, const Source &src) {
    for (size_t r = 0; r < q.rows; r += kRowsALaunch)
        any_row_kernel<Source, W><<<(unsigned)std::min(q.rows - r, kRowsALaunch), 64 * W, 0, s>>>(
            src, q.ptr, q.scale, r, (int)q.cols, (int)q8_frags(q.cols));
}

// Rows that fit a block's registers, in the block that they fill best: up to
// eight waves a row, with more loads in flight than four and more blocks a CU
// than sixteen (us with 4 / 8 / 16 waves: silu 2048 x 9728 44 / 38 / 53, rows
// 8192 x 4096 33 / 31 / 42; norm 8192 x 2560, which five fill, 49 / 52 / 60,
// five 48), and one wave for short ones (norm 8192 x 128 6.7 where four waves
// take 14.8, 8192 x 512 11.7 / 16.1, 8192 x 1024 21.0 / 19.6). Longer ones in
// parts of which only the values stay (us whole / in parts: norm 2048 x 8192
// 43.0 / 39.7, silu of it 31.7 / 30.9; silu 2048 x 12000 with sixteen waves
// 62.6, eight in parts 46.0; 1024 x 28000 by any_row 132, in parts 58).
//
// Each of the others against the next longer rows' block (us of the norm, and
// of silu, of 1024 rows; of 64 where it says so): <6, 1> 1536 columns 5.6 / 6.4,
// 6.0 / 6.5; <5, 2, 2> 5120 8.4 / 9.7, 11.7 / 13.2; <8, 3> 6144 of 64 rows 5.1 /
// 5.6, 5.7 / 6.1 (1024 rows 10.2 / 10.5, 13.8 both); <8, 3, 2> 12288 16.6 /
// 19.2, 24.2 / 26.2; <8, 2, 6> 24576 29.2 / 31.0, 48.2 / 49.9; <8, 2, 7> 28672
// 33.4 / 43.2, 56.3 / 66.3; <16, 2, 4> 32768 51.1 / 54.7, 71.8 / 77.5; <16, 2,
// 5> 40960 against any_row 61.8 / 86.1, 89.6 / 187. <8, 1> 2048 of 64 rows 4.05
// / 4.26, 4.2 / 4.5, but of 1024 rows 6.5 / 5.9, 7.0 / 6.9 with <5, 2>.
//
// Rows that have a CU each (up to 256) go the same ways (sixteen waves wait
// longer at their barriers than they save: norm of 4096 3.6 with eight, 4.3),
// but for 8193 to 10240 columns and 12289 to 20480: ten or sixteen waves take
// 1.05 to 1.2 times less for rows and 1.03 to 1.13 for silu, and the norm is up to 7%
// either way (64 rows, us eight waves / so: of 9728 4.2 / 3.9, silu 6.9 / 6.4,
// norm 5.9 both; of 20000 6.2 / 5.5, 10.2 / 9.5, 8.5 both; one row of 9728 2.75
// / 2.80, 4.7 / 4.9, 4.4 / 4.75). In a gated MLP of 1 to 128 tokens that is 0.1
// to 0.8 us a layer, with its weights from the caches or from memory (64 tokens
// of eight layers in turn, 9728 between, 51.1 / 50.6; 14336, 59.8 / 59.0; 20000,
// 70.4 / 69.6).
template <class Source>
hipError_t launch_rows(hipStream_t s, const th_q8 &q, const Source &src) {
    if (q.rows == 0) return hipSuccess;
    const size_t c = (q.cols + 255) / 256;
    if constexpr (!Source::kNt) {
        if (q.rows <= 256) {
            if (c > 32 && c <= 40) return launch_held<Source, 10, 2, 2>(s, q, src), hipGetLastError();
            if (c > 48 && c <= 64) return launch_held<Source, 16, 4>(s, q, src), hipGetLastError();
            if (c > 64 && c <= 80) return launch_held<Source, 16, 5>(s, q, src), hipGetLastError();
        }
    }
    if (c <= 1) launch_held<Source, 1, 1>(s, q, src);
    else if (c <= 2) launch_held<Source, 1, 2>(s, q, src);
    else if (c <= 4) launch_held<Source, 4, 1>(s, q, src);
    else if (c <= 6) launch_held<Source, 6, 1>(s, q, src);
    else if (c <= 8) launch_held<Source, 8, 1>(s, q, src);
    else if (c <= 10) launch_held<Source, 5, 2>(s, q, src);
    else if (c <= 16) launch_held<Source, 8, 2>(s, q, src);
    else if (c <= 20) launch_held<Source, 5, 2, 2>(s, q, src);
    else if (c <= 24) launch_held<Source, 8, 3>(s, q, src);
    else if (c <= 32) launch_held<Source, 8, 2, 2>(s, q, src);
    else if (c <= 40) launch_held<Source, 8, 5>(s, q, src);
    else if (c <= 48) launch_held<Source, 8, 3, 2>(s, q, src);
    else if (c <= 64) launch_held<Source, 8, 2, 4>(s, q, src);
    else if (c <= 80) launch_held<Source, 8, 2, 5>(s, q, src);
    else if (c <= 96) launch_held<Source, 8, 2, 6>(s, q, src);
    else if (c <= 112) launch_held<Source, 8, 2, 7>(s, q, src);
    else if (c <= 128) launch_held<Source, 16, 2, 4>(s, q, src);
    else if (c <= 160) launch_held<Source, 16, 2, 5>(s, q, src);
    else launch_any<Source, 16>(s, q, src);
    return hipGetLastError();
}

// Whether n inputs of q's shape are read past the caches' normal order.
bool past_caches(const th_q8 &q, size_t n) { return n * q.rows * q.cols * sizeof(float) >= kPastCaches; }

}  // namespace

hipError_t launch_quantize_q8(hipStream_t s, const th_q8 &q, const float *x) {
    return past_caches(q, 1) ? launch_rows(s, q, RowsSource<true>{x}) : launch_rows(s, q, RowsSource<false>{x});
}

hipError_t launch_quantize_weight_q8(hipStream_t s, const th_q8 &q, const uint16_t *w) {
    if (q.rows == 0) return hipSuccess;
    launch_any<WeightSource, 4>(s, q, WeightSource{w});
    return hipGetLastError();
}

hipError_t launch_add_rmsnorm_q8(hipStream_t s, float *x, const float *y, const th_q8 &q, const uint16_t *w, float eps) {
    return past_caches(q, y ? 2 : 1) ? launch_rows(s, q, NormSource<true>{x, y, w, eps})
                                     : launch_rows(s, q, NormSource<false>{x, y, w, eps});
}

hipError_t launch_silu_mul_q8(hipStream_t s, const th_q8 &q, const float *gate, const float *up) {
    return past_caches(q, 2) ? launch_rows(s, q, SiluSource<true>{gate, up})
                             : launch_rows(s, q, SiluSource<false>{gate, up});
}

hipError_t launch_reorder_q8(hipStream_t s, const th_q8 &q, int8_t *plain, size_t row0, size_t rows, bool in) {
    if (rows == 0) return hipSuccess;
    const unsigned blocks = (unsigned)((rows * ((q.cols + 15) / 16) + 255) / 256);
    const int cols = (int)q.cols, frags = (int)q8_frags(q.cols);
    if (in) reorder_kernel<true><<<blocks, 256, 0, s>>>(q.ptr, plain, row0, rows, cols, frags);
    else reorder_kernel<false><<<blocks, 256, 0, s>>>(q.ptr, plain, row0, rows, cols, frags);
    return hipGetLastError();
}

size_t dequantize_rows_a_launch(size_t cols) { return kBlocksALaunch / ((cols + 255) / 256) * 16; }

hipError_t launch_dequantize_q8(hipStream_t s, float *out, const th_q8 &q) {
    const size_t parts = (q.cols + 255) / 256, most = dequantize_rows_a_launch(q.cols), frags = q8_frags(q.cols);
    for (size_t r = 0; r < q.rows; r += most) {
        const size_t rows = std::min(q.rows - r, most);
        dequantize_kernel<<<(unsigned)(q8_blocks(rows) * parts), 256, 0, s>>>(
            out + r * q.cols, q.ptr + r / 16 * frags * 1024, q.scale + r, rows, (int)q.cols, (int)frags, (int)parts);
    }
    return hipGetLastError();
}

}  // namespace th

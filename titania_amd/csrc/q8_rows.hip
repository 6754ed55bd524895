// Rows in 8 bits: f32 rows, bf16 weights, rmsnorm(x + y) and silu(gate) * up
// as integers with a scale a row, and the values that such rows stand for.
//
// Of a row v with A = max |v|, the integers are those nearest to 127 v / A
// (ties to even) and the scale is A / 127 in f32; where that rounds to zero, so
// do the integers. The quotients are formed in
// 64 bits, so that the integers are the definition's whatever the launch. For
// rmsnorm, v_c = r x_c g_c with one positive r a row, which the quotients lose:
// 127 x_c g_c / max |x g|, whose products are exact in 64 bits.
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

// Four values from column c of a row, zeros past its end.
__device__ __forceinline__ void load4(const float *row, int c, int cols, float (&v)[4]);

// What a row is made of. value: the 64-bit value (of the norm without its
// factor r) at flat index i, column c. load: a thread's f32 values; kOff is how
// far they may be off, relative to the value. kMost: load has the largest
// 64-bit value itself.
struct RowsSource {
    static constexpr bool kNorm = false, kMost = false;
    static constexpr float kOff = 0;
    const float *x;
    __device__ double value(size_t i, size_t) const { return (double)x[i]; }
    template <int N, int T>
    __device__ void load(size_t row, int cols, float (&v)[N][4], double &, double &, int &) const {
#pragma unroll
        for (int k = 0; k < N; ++k) load4(x + row * cols, 4 * (threadIdx.x + T * k), cols, v[k]);
    }
};

struct WeightSource {
    static constexpr bool kNorm = false;
    const uint16_t *w;
    __device__ double value(size_t i, size_t) const { return (double)bf16_to_f32(w[i]); }
};

struct NormSource {
    static constexpr bool kNorm = true, kMost = true;
    static constexpr float kOff = 1.0f / (1 << 24);
    float *x;
    const float *y;
    const uint16_t *g;
    float eps;
    __device__ double value(size_t i, size_t c) const { return (double)x[i] * (double)bf16_to_f32(g[c]); }
    template <int N, int T>
    __device__ void load(size_t row, int cols, float (&v)[N][4], double &most, double &sum, int &) const;
};

struct SiluSource {
    static constexpr bool kNorm = false, kMost = false;
    // expf within 2 units in the last place (2^-23 each at most), the sum, the
    // quotient and the product within half of one.
    static constexpr float kOff = 3.5f / (1 << 23);
    const float *gate, *up;
    __device__ double value(size_t i, size_t) const {
        const double g = (double)gate[i];
        return g / (1.0 + exp(-g)) * (double)up[i];
    }
    template <int N, int T>
    __device__ void load(size_t row, int cols, float (&v)[N][4], double &, double &, int &odd) const {
        float u[N][4];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            load4(gate + row * cols, 4 * (threadIdx.x + T * k), cols, v[k]);
            load4(up + row * cols, 4 * (threadIdx.x + T * k), cols, u[k]);
        }
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                odd |= v[k][j] < -80.f;
                v[k][j] = silu(v[k][j]) * u[k][j];
            }
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

// The scale of a row whose largest value is most (of the norm: times a factor),
// and whether the row is marked instead.
template <class Source>
__device__ __forceinline__ float scale_of(const Source &src, double most, double sum, int cols, int &bad) {
    double top = most;
    if constexpr (Source::kNorm) top = most == 0 ? 0 : most / sqrt(sum / cols + (double)src.eps);
    const float s = (float)(top / 127.0);
    bad |= !(s <= FLT_MAX);
    return bad ? __builtin_nanf("") : s;
}

// A row in 64 bits, read once for its maximum and again for its integers: any
// row, by W waves.
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

template <class Source, int W>
__global__ __launch_bounds__(64 * W) void any_row_kernel(Source src, int8_t *__restrict__ q, float *__restrict__ scale,
                                                         int cols, int frags, bool add) {
    any_row<Source, W>(src, blockIdx.x, q, scale, cols, frags, add);
}

// Four f32 of a row, which starts at no more than 4-byte alignment.
struct __attribute__((packed, aligned(4))) Loose4 {
    float v[4];
};

__device__ __forceinline__ void load4(const float *row, int c, int cols, float (&v)[4]) {
    if (c + 4 <= cols) {
        const Loose4 l = *reinterpret_cast<const Loose4 *>(row + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = l.v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = c + j < cols ? row[c + j] : 0.f;
    }
}

template <int N, int T>
__device__ void NormSource::load(size_t row, int cols, float (&v)[N][4], double &most, double &sum, int &odd) const {
    float u[N][4];
    alignas(8) uint16_t gain[N][4];
    float *xr = x + row * cols;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int c = 4 * (threadIdx.x + T * k);
        load4(xr, c, cols, v[k]);
        if (y) load4(y + row * cols, c, cols, u[k]);
        if (c + 4 <= cols) {
            *reinterpret_cast<uint2 *>(gain[k]) = *reinterpret_cast<const uint2 *>(g + c);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) gain[k][j] = c + j < cols ? g[c + j] : 0;
        }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int c = 4 * (threadIdx.x + T * k);
        if (y) {
            Loose4 l;
#pragma unroll
            for (int j = 0; j < 4; ++j) l.v[j] = v[k][j] += u[k][j];
            if (c + 4 <= cols) {
                *reinterpret_cast<Loose4 *>(xr + c) = l;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < cols) xr[c + j] = l.v[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double d = (double)v[k][j];
            const float f = bf16_to_f32(gain[k][j]);
            odd |= !(fabsf(v[k][j]) <= FLT_MAX);
            sum = fma(d, d, sum);
            most = fmax(most, fabs(d * (double)f));
            v[k][j] *= f;
        }
    }
}

// Rows of up to 256 W N columns, one block of W waves a row, N times four
// columns a thread, held in registers, so that the row is read once.
//
// Bound by memory. What 64 bits decide is found in 32 first: a value's f32 is
// off by at most Source::kOff of it and the quotient by 127 times that and two
// roundings more, so only values within twice that of the largest are compared
// in 64 bits, and only quotients within 127 kNear of a border are formed again
// (3 in 10000 for silu). Rows on which f32 does not hold what 64 bits do
// (values past 1e38 or not finite, none as large as 1e-30, arguments whose
// exponential overflows) are taken by any_row.
template <class Source, int W, int N>
__global__ __launch_bounds__(64 * W) void rows_kernel(Source src, int8_t *__restrict__ q, float *__restrict__ scale,
                                                      size_t rows, int cols, int frags, bool grouped) {
    constexpr int T = 64 * W;
    constexpr float kNear = Source::kOff + 3.0f / (1 << 24);
    __shared__ Reduced<W> sh[2];
    const size_t row = row_of_block(blockIdx.x, grouped);
    if (row >= rows) return;
    float v[N][4];
    double most = 0, sum = 0;
    int odd = 0;
    src.template load<N, T>(row, cols, v, most, sum, odd);
    float m = 0;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float a = fabsf(v[k][j]);
            odd |= !(a < 1e38f);
            m = fmaxf(m, a);
        }
    if constexpr (!Source::kMost) most = m;
    reduce(sh[0], most, sum, odd);
    odd |= most < 1e-30;
    if (odd) {
        any_row<Source, W>(src, row, q, scale, cols, frags, false);
        return;
    }
    if constexpr (!Source::kMost && Source::kOff > 0) {
        const float reach = (float)most * (1 - 2 * Source::kOff - 1.0f / (1 << 23));
        double exact = 0, unused = 0;
        int none = 0;
        if (m >= reach) {
#pragma unroll
            for (int k = 0; k < N; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (fabsf(v[k][j]) >= reach) {
                        const int c = 4 * (threadIdx.x + T * k) + j;
                        exact = fmax(exact, fabs(src.value(row * cols + c, c)));
                    }
        }
        reduce(sh[1], exact, unused, none);
        most = exact;
    }
    int bad = 0;
    const float s = scale_of(src, most, sum, cols, bad);
    if (threadIdx.x == 0) scale[row] = s;
    const double inv = 127.0 / most;
    const float inv32 = (float)inv;
    char4 *out = reinterpret_cast<char4 *>(q);
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int c0 = 4 * (threadIdx.x + T * k);
        if (c0 >= cols) break;
        int n[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float t = v[k][j] * inv32, r = rintf(t);
            n[j] = (int)r;
            if (fabsf(fabsf(t - r) - 0.5f) < 127 * kNear && c0 + j < cols)
                n[j] = nearest(src.value(row * cols + c0 + j, c0 + j), most, inv);
            if (bad || s == 0) n[j] = 0;
        }
        out[q8_at(row, c0, frags) / 4] = make_char4((char)n[0], (char)n[1], (char)n[2], (char)n[3]);
    }
}

// A block a 16 rows x 256 columns: four rows of four columns a thread.
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
        const Loose4 l{{v[i].x * s[i], v[i].y * s[i], v[i].z * s[i], v[i].w * s[i]}};
        if (c + 4 <= cols) {
            *reinterpret_cast<Loose4 *>(o) = l;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < cols) o[j] = l.v[j];
        }
    }
}

template <class Source, int W, int N>
void launch_held(hipStream_t s, const th_q8 &q, const Source &src) {
    const bool grouped = q.rows >= 128;
    const size_t blocks = grouped ? (q.rows + 127) / 128 * 128 : q.rows;
    rows_kernel<Source, W, N><<<(unsigned)blocks, 64 * W, 0, s>>>(src, q.ptr, q.scale, q.rows, (int)q.cols,
                                                                  (int)q8_frags(q.cols), grouped);
}

// Rows that fit a block's registers: few of them with 16 waves a row, which
// have it sooner, many with 4, of which a CU runs several rows at once.
template <class Source>
hipError_t launch_rows(hipStream_t s, const th_q8 &q, const Source &src) {
    if (q.rows == 0) return hipSuccess;
    const size_t c = q.cols;
    if (q.rows > 256 && c <= 10240) {
        if (c <= 1024) launch_held<Source, 4, 1>(s, q, src);
        else if (c <= 2048) launch_held<Source, 4, 2>(s, q, src);
        else if (c <= 3 * 1024) launch_held<Source, 4, 3>(s, q, src);
        else if (c <= 4096) launch_held<Source, 4, 4>(s, q, src);
        else if (c <= 6 * 1024) launch_held<Source, 4, 6>(s, q, src);
        else if (c <= 8192) launch_held<Source, 4, 8>(s, q, src);
        else launch_held<Source, 4, 10>(s, q, src);
    } else if (c <= 20480) {
        if (c <= 1024) launch_held<Source, 4, 1>(s, q, src);
        else if (c <= 4096) launch_held<Source, 16, 1>(s, q, src);
        else if (c <= 8192) launch_held<Source, 16, 2>(s, q, src);
        else if (c <= 12288) launch_held<Source, 16, 3>(s, q, src);
        else launch_held<Source, 16, 5>(s, q, src);
    } else {
        any_row_kernel<Source, 16><<<(unsigned)q.rows, 1024, 0, s>>>(src, q.ptr, q.scale, (int)q.cols,
                                                                     (int)q8_frags(q.cols), true);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_quantize_q8(hipStream_t s, const th_q8 &q, const float *x) { return launch_rows(s, q, RowsSource{x}); }

hipError_t launch_quantize_weight_q8(hipStream_t s, const th_q8 &q, const uint16_t *w) {
    if (q.rows == 0) return hipSuccess;
    any_row_kernel<WeightSource, 4><<<(unsigned)q.rows, 256, 0, s>>>(WeightSource{w}, q.ptr, q.scale, (int)q.cols,
                                                                     (int)q8_frags(q.cols), true);
    return hipGetLastError();
}

hipError_t launch_add_rmsnorm_q8(hipStream_t s, float *x, const float *y, const th_q8 &q, const uint16_t *w, float eps) {
    return launch_rows(s, q, NormSource{x, y, w, eps});
}

hipError_t launch_silu_mul_q8(hipStream_t s, const th_q8 &q, const float *gate, const float *up) {
    return launch_rows(s, q, SiluSource{gate, up});
}

hipError_t launch_dequantize_q8(hipStream_t s, float *out, const th_q8 &q) {
    if (q.rows == 0) return hipSuccess;
    const size_t parts = (q.cols + 255) / 256;
    dequantize_kernel<<<(unsigned)(q8_blocks(q.rows) * parts), 256, 0, s>>>(out, q.ptr, q.scale, q.rows, (int)q.cols,
                                                                            (int)q8_frags(q.cols), (int)parts);
    return hipGetLastError();
}

}  // namespace th

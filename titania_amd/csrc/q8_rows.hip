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

constexpr int kThreads = 256;

// The nearest integer to 127 v / most. inv: 127 / most. v * inv is off by at
// most 127 * 2^-52, so only what lies within 1e-12 of a border is divided.
__device__ __forceinline__ int nearest(double v, double most, double inv) {
    double t = v * inv;
    if (fabs(fabs(t - trunc(t)) - 0.5) < 1e-12) t = v * 127.0 / most;
    return (int)rint(t);
}

struct RowsSource {
    const float *x;
    __device__ double value(size_t i, size_t) const { return (double)x[i]; }
};

struct WeightSource {
    const uint16_t *w;
    __device__ double value(size_t i, size_t) const { return (double)bf16_to_f32(w[i]); }
};

struct NormSource {
    float *x;
    const float *y;
    const uint16_t *g;
    float eps;
    __device__ double value(size_t i, size_t c) const { return (double)x[i] * (double)bf16_to_f32(g[c]); }
};

struct SiluSource {
    const float *gate, *up;
    __device__ double value(size_t i, size_t) const {
        const double g = (double)gate[i];
        return g / (1.0 + exp(-g)) * (double)up[i];
    }
};

// One block a row, the row read once for its maximum and again for its integers.
template <class Source>
__global__ __launch_bounds__(kThreads) void rows_kernel(Source src, int8_t *__restrict__ q, float *__restrict__ scale,
                                                        int cols, int frags) {
    constexpr bool kNorm = __is_same(Source, NormSource);
    __shared__ double red_max[kThreads / 64], red_sum[kThreads / 64];
    __shared__ int red_bad[kThreads / 64];
    const size_t row = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double most = 0, sum = 0;
    int bad = 0;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
        const size_t i = row * cols + c;
        if constexpr (kNorm) {
            float v = src.x[i];
            if (src.y) src.x[i] = v += src.y[i];
            sum += (double)v * (double)v;
        }
        const double v = fabs(src.value(i, c));
        bad |= !(v <= DBL_MAX);
        most = fmax(most, v);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        most = fmax(most, __shfl_xor(most, o, 64));
        sum += __shfl_xor(sum, o, 64);
    }
    bad = __any(bad);
    if (lane == 0) {
        red_max[wave] = most;
        red_sum[wave] = sum;
        red_bad[wave] = bad;
    }
    __syncthreads();
    most = sum = 0;
    bad = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        most = fmax(most, red_max[w]);
        sum += red_sum[w];
        bad |= red_bad[w];
    }
    double top = most;
    if constexpr (kNorm) top = most == 0 ? 0 : most / sqrt(sum / cols + (double)src.eps);
    float s = (float)(top / 127.0);
    if (bad || !(s <= FLT_MAX)) s = __builtin_nanf(""), bad = 1;
    if (threadIdx.x == 0) scale[row] = s;
    const double inv = 127.0 / most;
    for (int c = threadIdx.x; c < cols; c += kThreads) {
        const size_t i = row * cols + c;
        q[q8_at(row, c, frags)] = bad || s == 0 ? 0 : (int8_t)nearest(src.value(i, c), most, inv);
    }
}

// A block a 16 rows x 256 columns, 4 columns a thread.
__global__ __launch_bounds__(kThreads) void dequantize_kernel(float *__restrict__ out, const int8_t *__restrict__ q,
                                                              const float *__restrict__ scale, size_t rows, int cols,
                                                              int frags) {
    const int c = ((int)blockIdx.y * 64 + (threadIdx.x & 63)) * 4;
    if (c >= cols) return;
    for (int r = threadIdx.x >> 6; r < 16; r += kThreads / 64) {
        const size_t row = (size_t)blockIdx.x * 16 + r;
        if (row >= rows) return;
        const float s = scale[row];
        const char4 v = *reinterpret_cast<const char4 *>(q + q8_at(row, c, frags));
        float *o = out + row * cols + c;
        if (cols % 4 == 0) {
            *reinterpret_cast<float4 *>(o) = make_float4(v.x * s, v.y * s, v.z * s, v.w * s);
        } else {
            o[0] = v.x * s;
            if (c + 1 < cols) o[1] = v.y * s;
            if (c + 2 < cols) o[2] = v.z * s;
            if (c + 3 < cols) o[3] = v.w * s;
        }
    }
}

template <class Source>
hipError_t launch_rows(hipStream_t s, const th_q8 &q, const Source &src) {
    if (q.rows == 0) return hipSuccess;
    rows_kernel<<<(unsigned)q.rows, kThreads, 0, s>>>(src, q.ptr, q.scale, (int)q.cols, (int)q8_frags(q.cols));
    return hipGetLastError();
}

}  // namespace

hipError_t launch_quantize_q8(hipStream_t s, const th_q8 &q, const float *x) { return launch_rows(s, q, RowsSource{x}); }

hipError_t launch_quantize_weight_q8(hipStream_t s, const th_q8 &q, const uint16_t *w) {
    return launch_rows(s, q, WeightSource{w});
}

hipError_t launch_add_rmsnorm_q8(hipStream_t s, float *x, const float *y, const th_q8 &q, const uint16_t *w, float eps) {
    return launch_rows(s, q, NormSource{x, y, w, eps});
}

hipError_t launch_silu_mul_q8(hipStream_t s, const th_q8 &q, const float *gate, const float *up) {
    return launch_rows(s, q, SiluSource{gate, up});
}

hipError_t launch_dequantize_q8(hipStream_t s, float *out, const th_q8 &q) {
    if (q.rows == 0) return hipSuccess;
    const dim3 grid((unsigned)q8_blocks(q.rows), (unsigned)((q.cols + 255) / 256));
    dequantize_kernel<<<grid, kThreads, 0, s>>>(out, q.ptr, q.scale, q.rows, (int)q.cols, (int)q8_frags(q.cols));
    return hipGetLastError();
}

}  // namespace th

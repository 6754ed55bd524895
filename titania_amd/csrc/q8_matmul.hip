// Products of 8-bit rows on the matrix cores:
// out[t][r] = x.scale[t] w.scale[r] sum_k x[t][k] w[r][k].
//
// The sums are exact (32-bit integers), so that neither the order nor a split
// of K changes a result; then one conversion to f32 and two products.
#include "device_util.h"
#include "q8.h"

namespace th {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

struct Args {
    const int8_t *w, *x;
    const float *w_scale, *x_scale;
    float *out;
    int n, rows, frags;
};

// A wave a 16 rows x 16 tokens: the weights' fragment is the first operand, so
// lane l ends with rows 4 (l / 16) .. + 3 of token l % 16.
__global__ __launch_bounds__(256) void matmul_kernel(Args a) {
    const int lane = threadIdx.x & 63;
    const int quads = (a.rows + 63) / 64;
    const int rb = (int)(blockIdx.x % quads) * 4 + (threadIdx.x >> 6), tb = blockIdx.x / quads;
    if (rb * 16 >= a.rows) return;
    const i32x4 *w = reinterpret_cast<const i32x4 *>(a.w) + (size_t)rb * a.frags * 64 + lane;
    const i32x4 *x = reinterpret_cast<const i32x4 *>(a.x) + (size_t)tb * a.frags * 64 + lane;
    i32x4 sum = {0, 0, 0, 0};
    for (int f = 0; f < a.frags; ++f)
        sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[(size_t)f * 64], x[(size_t)f * 64], sum, 0, 0, 0);
    const int t = tb * 16 + (lane & 15), r = rb * 16 + (lane >> 4) * 4;
    if (t >= a.n) return;
    const float xs = a.x_scale[t];
    for (int i = 0; i < 4; ++i)
        if (r + i < a.rows) a.out[(size_t)t * a.rows + r + i] = (float)sum[i] * xs * a.w_scale[r + i];
}

}  // namespace

hipError_t launch_matmul_q8(hipStream_t s, float *out, const th_q8 &w, const th_q8 &x) {
    if (x.rows == 0 || w.rows == 0) return hipSuccess;
    const Args a{w.ptr, x.ptr, w.scale, x.scale, out, (int)x.rows, (int)w.rows, (int)q8_frags(w.cols)};
    matmul_kernel<<<(unsigned)((w.rows + 63) / 64 * q8_blocks(x.rows)), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace th

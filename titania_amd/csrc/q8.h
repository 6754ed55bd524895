// 8-bit rows (th_q8): their layout, and the launchers of their kernels.
#pragma once

#include <algorithm>

#include "common.h"
#include "gemm.h"

// Rows of 8-bit integers with an f32 scale each. A wave's matrix-core operand
// of 16 rows x 64 columns (a fragment) is 1 KB of consecutive memory, lane
// l = row % 16 + 16 * (column % 64 / 16) having 16 consecutive columns, so
// that operands are loaded, staged in LDS and read back 16 consecutive bytes a
// lane, with neither a transposition nor a bank conflict. The fragments of 16
// rows lie side by side. Columns past `cols` of a row are zero, always.
struct th_q8 {
    int8_t *ptr = nullptr;
    float *scale = nullptr;  // behind the integers, in the same allocation
    size_t rows = 0;         // current rows
    size_t cap = 0;          // rows it was allocated with
    size_t cols = 0;
    int ordinal = 0;         // the GPU that holds it
};

namespace th {

// Sums of cols products of two 8-bit integers stay below 2^31.
constexpr size_t kQ8MaxCols = 131071;
// Of what fits 288 GB, a product's launch then has fewer than 2^32 threads.
constexpr size_t kQ8MaxRows = (size_t)1 << 25;

// The device's block of partials, which calls use in the stream's order.
constexpr size_t kQ8PartBytes = std::max(kPartFloats, kAttnRoundFloats) * sizeof(float);

// Fragments of a row block: an even number, for kernels that step by 128 columns.
constexpr size_t q8_frags(size_t cols) { return (cols + 127) / 128 * 2; }
constexpr size_t q8_blocks(size_t rows) { return (rows + 15) / 16; }
// Byte of (row, col) in a matrix of `frags` fragments a row block.
__host__ __device__ constexpr size_t q8_at(size_t row, size_t col, size_t frags) {
    return ((row >> 4) * frags + (col >> 6)) * 1024 + ((row & 15) + (col >> 4 & 3) * 16) * 16 + (col & 15);
}

// Rows row0 .. of q from `rows` of them row-major in plain (in), or to there.
hipError_t launch_reorder_q8(hipStream_t s, const th_q8 &q, int8_t *plain, size_t row0, size_t rows, bool in);
// q = 8-bit rows of x [rows][cols] (f32, or bf16 weights).
hipError_t launch_quantize_q8(hipStream_t s, const th_q8 &q, const float *x);
hipError_t launch_quantize_weight_q8(hipStream_t s, const th_q8 &q, const uint16_t *w);
// out [rows][cols] = the values that q stands for.
hipError_t launch_dequantize_q8(hipStream_t s, float *out, const th_q8 &q);
// The rows that one launch of it takes, a multiple of 16.
size_t dequantize_rows_a_launch(size_t cols);
// x += y (unless y is null), q = 8-bit rows of rmsnorm(x).
hipError_t launch_add_rmsnorm_q8(hipStream_t s, float *x, const float *y, const th_q8 &q, const uint16_t *w, float eps);
// q = 8-bit rows of silu(gate) * up.
hipError_t launch_silu_mul_q8(hipStream_t s, const th_q8 &q, const float *gate, const float *up);
// out[t * w.rows + r] = x.scale[t] w.scale[r] sum_k x[t][k] w[r][k]. Where it
// splits K, the sums of the parts go to part (part_len long).
hipError_t launch_matmul_q8(hipStream_t s, float *out, const th_q8 &w, const th_q8 &x, int *part, size_t part_len);
// Which of its variants it takes (the few-token kernel's, then the tiles'), and
// the parts of K.
int matmul_q8_variant(size_t n, size_t rows, size_t cols, size_t part_len, int *ksplit);

// Four f32 at any multiple of 4 bytes: the memory path takes 16 bytes at any of
// them, as one access where the type says so.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// Stores the first `left` of four values (all, if more are left). NT: past the
// caches' normal order, for results larger than they are.
template <bool NT = false>
__device__ __forceinline__ void store4(float *o, f32x4_any v, int left) {
    if (left >= 4) {
        if (NT) __builtin_nontemporal_store(v, reinterpret_cast<f32x4_any *>(o));
        else *reinterpret_cast<f32x4_any *>(o) = v;
    } else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < left) o[i] = v[i];
    }
}

}  // namespace th

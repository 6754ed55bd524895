// The C ABI's 8-bit rows (th_q8): handles, host copies and argument checks.
#include <algorithm>
#include <new>

#include "common.h"
#include "q8.h"

using th::fail;

namespace {

// Rows in another GPU's memory are refused.
#define TH_Q8_HERE(dev, q) \
    TH_REQUIRE((q)->ordinal == (dev)->ordinal, "8-bit rows of GPU %d on GPU %d", (q)->ordinal, (dev)->ordinal)

#define TH_Q8_CURRENT(dev)     \
    th::Current current_(dev); \
    TH_HIP(current_.error)

// Bytes of the integers of `rows` rows.
size_t value_bytes(size_t rows, size_t cols) { return th::q8_blocks(rows) * th::q8_frags(cols) * 1024; }

}  // namespace

extern "C" {

int th_q8_alloc(th_device *dev, size_t rows, size_t cols, th_q8 **out) {
    TH_REQUIRE(dev && out, "th_q8_alloc: null argument");
    TH_NOT_CAPTURING(dev, "th_q8_alloc");
    TH_REQUIRE(cols > 0 && cols <= th::kQ8MaxCols, "8-bit rows of %zu columns: 1 to %zu", cols, th::kQ8MaxCols);
    TH_REQUIRE(rows <= th::kQ8MaxRows, "%zu 8-bit rows: at most %zu", rows, th::kQ8MaxRows);
    TH_Q8_CURRENT(dev);
    auto *q = new (std::nothrow) th_q8();
    if (!q) return fail(TH_ERR_NOMEM, "out of host memory");
    const size_t values = value_bytes(rows, cols), bytes = values + std::max<size_t>(th::q8_blocks(rows) * 64, 64);
    hipError_t e = hipMalloc(&q->ptr, bytes);
    if (e == hipSuccess) e = hipMemsetAsync(q->ptr, 0, bytes, dev->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(dev->stream);
    if (e != hipSuccess) {
        (void)hipGetLastError();  // reported here, not by the next launch
        if (q->ptr) (void)hipFree(q->ptr);
        delete q;
        return fail(e == hipErrorOutOfMemory ? TH_ERR_NOMEM : TH_ERR_HIP, "alloc of %zu x %zu 8-bit rows failed: %s",
                    rows, cols, hipGetErrorString(e));
    }
    q->scale = reinterpret_cast<float *>(q->ptr + values);
    q->rows = q->cap = rows;
    q->cols = cols;
    q->ordinal = dev->ordinal;
    *out = q;
    return TH_OK;
}

void th_q8_free(th_device *dev, th_q8 *q) {
    if (!q) return;
    if (dev && dev->capturing) {  // the handle stays valid: free it after th_graph_end
        fail(TH_ERR_INVALID, "th_q8_free cannot run while the device's stream is being captured");
        return;
    }
    if (dev) (void)hipStreamSynchronize(dev->stream);
    if (q->ptr) (void)hipFree(q->ptr);
    delete q;
}

int th_q8_shape(const th_q8 *q, size_t *rows, size_t *cols) {
    TH_REQUIRE(q && rows && cols, "th_q8_shape: null argument");
    *rows = q->rows;
    *cols = q->cols;
    return TH_OK;
}

int th_q8_resize(th_device *dev, th_q8 *q, size_t rows) {
    TH_REQUIRE(dev && q, "th_q8_resize: null argument");
    TH_REQUIRE(rows <= q->cap, "%zu 8-bit rows can't hold %zu", q->cap, rows);
    q->rows = rows;
    return TH_OK;
}

int th_q8_read(th_device *dev, const th_q8 *q, int8_t *values, float *scales) {
    TH_REQUIRE(dev && q, "th_q8_read: null argument");
    TH_NOT_CAPTURING(dev, "th_q8_read");
    TH_REQUIRE(q->rows == 0 || (values && scales), "th_q8_read: null output");
    TH_Q8_HERE(dev, q);
    TH_Q8_CURRENT(dev);
    // Through the device's block of partials, as many rows at a time as it holds.
    auto *plain = reinterpret_cast<int8_t *>(dev->part);
    const size_t most = th::kQ8PartBytes / q->cols;
    hipError_t e = hipSuccess;
    for (size_t r = 0; r < q->rows && e == hipSuccess; r += most) {
        const size_t n = std::min(most, q->rows - r);
        e = th::launch_reorder_q8(dev->stream, *q, plain, r, n, false);
        if (e == hipSuccess)
            e = hipMemcpyAsync(values + r * q->cols, plain, n * q->cols, hipMemcpyDeviceToHost, dev->stream);
    }
    if (e == hipSuccess && q->rows)
        e = hipMemcpyAsync(scales, q->scale, q->rows * sizeof(float), hipMemcpyDeviceToHost, dev->stream);
    const hipError_t done = hipStreamSynchronize(dev->stream);
    if (e == hipSuccess) e = done;
    if (e != hipSuccess) return fail(TH_ERR_HIP, "reading 8-bit rows failed: %s", hipGetErrorString(e));
    return TH_OK;
}

int th_q8_write(th_device *dev, th_q8 *q, const int8_t *values, const float *scales) {
    TH_REQUIRE(dev && q, "th_q8_write: null argument");
    TH_NOT_CAPTURING(dev, "th_q8_write");
    TH_REQUIRE(q->rows == 0 || (values && scales), "th_q8_write: null data");
    TH_Q8_HERE(dev, q);
    TH_Q8_CURRENT(dev);
    auto *plain = reinterpret_cast<int8_t *>(dev->part);
    const size_t most = th::kQ8PartBytes / q->cols;
    hipError_t e = hipSuccess;
    for (size_t r = 0; r < q->rows && e == hipSuccess; r += most) {
        const size_t n = std::min(most, q->rows - r);
        e = hipMemcpyAsync(plain, values + r * q->cols, n * q->cols, hipMemcpyHostToDevice, dev->stream);
        if (e == hipSuccess) e = th::launch_reorder_q8(dev->stream, *q, plain, r, n, true);
    }
    if (e == hipSuccess && q->rows)
        e = hipMemcpyAsync(q->scale, scales, q->rows * sizeof(float), hipMemcpyHostToDevice, dev->stream);
    const hipError_t done = hipStreamSynchronize(dev->stream);  // the host's arrays are read until then
    if (e == hipSuccess) e = done;
    if (e != hipSuccess) return fail(TH_ERR_HIP, "writing 8-bit rows failed: %s", hipGetErrorString(e));
    return TH_OK;
}

int th_quantize_q8(th_device *dev, th_q8 *q, const th_buffer *x) {
    TH_REQUIRE(dev && q && x, "th_quantize_q8: null argument");
    TH_REQUIRE(x->len == q->rows * q->cols, "x holds %zu activations, not %zu rows of %zu", x->len, q->rows, q->cols);
    TH_Q8_HERE(dev, q);
    TH_Q8_CURRENT(dev);
    TH_HIP(th::launch_quantize_q8(dev->stream, *q, x->ptr));
    return TH_OK;
}

int th_quantize_weight_q8(th_device *dev, th_q8 *q, const th_weight *w) {
    TH_REQUIRE(dev && q && w, "th_quantize_weight_q8: null argument");
    TH_REQUIRE(w->ndim == 2 && w->shape[0] == q->rows && w->shape[1] == q->cols,
               "the weight is not a matrix of %zu rows of %zu", q->rows, q->cols);
    TH_Q8_HERE(dev, q);
    TH_Q8_CURRENT(dev);
    TH_HIP(th::launch_quantize_weight_q8(dev->stream, *q, w->ptr));
    return TH_OK;
}

int th_dequantize_q8(th_device *dev, th_buffer *out, const th_q8 *q) {
    TH_REQUIRE(dev && out && q, "th_dequantize_q8: null argument");
    TH_REQUIRE(out->len == q->rows * q->cols, "out holds %zu activations, not %zu rows of %zu", out->len, q->rows,
               q->cols);
    TH_Q8_HERE(dev, q);
    TH_Q8_CURRENT(dev);
    TH_HIP(th::launch_dequantize_q8(dev->stream, out->ptr, *q));
    return TH_OK;
}

int th_add_rmsnorm_q8(th_device *dev, th_buffer *x, const th_buffer *y, th_q8 *q, const th_weight *w, float eps) {
    TH_REQUIRE(dev && x && q && w, "th_add_rmsnorm_q8: null argument");
    TH_REQUIRE(w->numel == q->cols, "%zu gains for rows of %zu", w->numel, q->cols);
    TH_REQUIRE(x->len == q->rows * q->cols, "x holds %zu activations, not %zu rows of %zu", x->len, q->rows, q->cols);
    TH_REQUIRE(!y || y->len >= x->len, "y holds %zu activations, x %zu", y ? y->len : 0, x->len);
    TH_REQUIRE(!y || y->ptr != x->ptr, "y must not alias x");
    TH_Q8_HERE(dev, q);
    TH_Q8_CURRENT(dev);
    TH_HIP(th::launch_add_rmsnorm_q8(dev->stream, x->ptr, y ? y->ptr : nullptr, *q, w->ptr, eps));
    return TH_OK;
}

int th_silu_mul_q8(th_device *dev, th_q8 *q, const th_buffer *gate, const th_buffer *up) {
    TH_REQUIRE(dev && q && gate && up, "th_silu_mul_q8: null argument");
    TH_REQUIRE(gate->len == q->rows * q->cols && up->len == gate->len,
               "gate and up hold %zu and %zu activations, not %zu rows of %zu", gate->len, up->len, q->rows, q->cols);
    TH_Q8_HERE(dev, q);
    TH_Q8_CURRENT(dev);
    TH_HIP(th::launch_silu_mul_q8(dev->stream, *q, gate->ptr, up->ptr));
    return TH_OK;
}

int th_matmul_q8(th_device *dev, th_buffer *out, const th_q8 *w, const th_q8 *x) {
    TH_REQUIRE(dev && out && w && x, "th_matmul_q8: null argument");
    TH_REQUIRE(x->cols == w->cols, "rows of %zu against weights of %zu columns", x->cols, w->cols);
    TH_REQUIRE(out->len == x->rows * w->rows, "out holds %zu activations, not %zu tokens x %zu rows", out->len, x->rows,
               w->rows);
    TH_Q8_HERE(dev, w);
    TH_Q8_HERE(dev, x);
    TH_Q8_CURRENT(dev);
    TH_HIP(th::launch_matmul_q8(dev->stream, out->ptr, *w, *x, reinterpret_cast<int *>(dev->part),
                                th::kQ8PartBytes / sizeof(int)));
    return TH_OK;
}

}  // extern "C"

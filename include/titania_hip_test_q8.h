/*
 * titania_hip_test_q8.h: test-only entry points about the 8-bit rows of
 * titania_hip.h. They answer from sizes alone, what a call launches, need no GPU
 * and are not part of the Device boundary.
 */
#ifndef TITANIA_HIP_TEST_Q8_H
#define TITANIA_HIP_TEST_Q8_H

#include "titania_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The threads of the largest launch of th_dequantize_q8. */
TH_API int th_test_dequantize_q8_threads(size_t rows, size_t cols, size_t *threads);

/* What th_matmul_q8 takes for n tokens: *variant, the few-token kernel's seven
 * first, then the tiles' eleven, in the order of their tables, and *ksplit, the
 * parts of K. */
TH_API int th_test_matmul_q8_variant(size_t n, size_t rows, size_t cols, int *variant, int *ksplit);

#ifdef __cplusplus
}
#endif

#endif

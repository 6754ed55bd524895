/*
 * titania_hip_test_paged.h: for tests/test_paged*.py alone: the attention's
 * kernels where a plan would take others, how th_batch_accept cuts its rows, and
 * what th_batch_set checks and plans, without a GPU.
 */
#ifndef TITANIA_HIP_TEST_PAGED_H
#define TITANIA_HIP_TEST_PAGED_H

#include "titania_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Later sets plan for these kernels (a bit each: tiles of 16 rows, always, of 128
 * and of 256), each for the sequences of 1 to 16, to 128 and of more rows, and for
 * the others the next there is, whatever would be fastest. */
TH_API int th_test_batch_classes(th_batch *batch, unsigned classes);

/* How th_batch_accept cuts `rows` rows of `cols` logits: rows a launch, parts a
 * row, values a part (the last one's are fewer). */
TH_API int th_test_accept_parts(size_t rows, size_t cols, size_t *rows_at_once, size_t *splits, size_t *part);

/* th_batch_set for a batch of shape {pages, page_len, n_kv_heads, head_dim,
 * kv_dtype, n_heads, max_seqs, max_tokens, max_pages} whose captured calls
 * launch `classes` of the attention's kernels (a bit each, the first always)
 * and captured_tokens tokens, with a table of captured_positions. Writes the tokens [n][4] (row of the cache,
 * position, sequence, place), what those of trees see [n][4], the attention's
 * items [..][9] (the sequence's first token, tokens, context, first page,
 * whether it is a tree; first row, first position, end, first slab), its joins
 * [..][6] (first token, rows, first row, first slab, parts, slabs of a part),
 * of which *n_items and *n_joins say how many there is room for, then are, and
 * the classes' first items [4]. */
TH_API int th_test_batch_set(const size_t *shape, unsigned classes, size_t captured_tokens, size_t captured_positions,
                             size_t n_seqs, const uint32_t *context, const uint32_t *n_new, const uint32_t *pages, size_t n_pages,
                             const int32_t *parents, uint32_t *tokens, uint64_t *tree, uint32_t *items, size_t *n_items,
                             uint32_t *joins, size_t *n_joins, uint32_t *first);

/* What a set that the GPU fails leaves of a batch of this shape: sequences,
 * tokens, pages and positions of the host, then of what launches are counted by
 * sequences, tokens, joins, their rows and items: nine numbers. Returns
 * th_batch_set's error. */
TH_API int th_test_batch_set_failed(const size_t *shape, size_t n_seqs, const uint32_t *context, const uint32_t *n_new,
                                    const uint32_t *pages, size_t n_pages, size_t *left);

#ifdef __cplusplus
}
#endif

#endif /* TITANIA_HIP_TEST_PAGED_H */

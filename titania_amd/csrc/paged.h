// Paged caches (th_paged) and the batches that use them (th_batch): their
// layout in memory, and the launchers of their kernels.
#pragma once

#include <algorithm>

#include "common.h"

// One layer's keys and values of many sequences, in pages of `page_len`
// positions: [page][keys, values][kv head][row][head_dim], f32 or bf16, so that
// what an attention of one KV head reads of a page is consecutive memory.
struct th_paged {
    void *ptr = nullptr;
    size_t pages = 0, page_len = 0, n_kv_heads = 0, head_dim = 0;
    int kv_dtype = TH_KV_F32;
    int ordinal = 0;  // the GPU that holds it
};

namespace th {

constexpr size_t kTreeTokens = 256;  // drafted tokens of one sequence's tree
constexpr int kTreeWords = (int)kTreeTokens / 64;
constexpr size_t kPagedMaxGroup = 16;  // query heads per KV head
constexpr size_t kMostPositions = (size_t)1 << 30;  // of a sequence, whose kernels count in 32 bits

// What the kernels read of a batch. A token: the row of the cache that it is
// written to (page * page_len + row) and the position of its rotation.
struct TokenAt {
    uint32_t slot, pos;
};
// A sequence: its first token, its tokens, the positions before them, where
// its pages begin in the list of pages, and whether its tokens form a tree
// (they see what `tree` says) or a chain.
struct SeqAt {
    uint32_t token0, n_new, context, page0, is_tree;
};
// The attention's work, planned once a step for all layers: rows (token, query
// head of the group) [row0, row0 + the class's tile) of a sequence over its
// positions [k0, k1), for each KV head. Where a tile's positions are split,
// `part` is the first slab of its partials (kNoPart: none).
constexpr int kClasses = 3;
constexpr int kClassRows[kClasses] = {16, 128, 256};
constexpr uint32_t kNoPart = 0xffffffffu;
// With its sequence's fields, so that a block's chain of loads is one shorter.
struct ItemAt {
    SeqAt seq;
    uint32_t row0, k0, k1, part;
};
// A split tile's rows, of the sequence at token0: `n_parts` items, each with
// `slabs` slabs for each KV head.
struct JoinAt {
    uint32_t token0, rows, row0, part, n_parts, slabs;
};
// A slab: 16 rows' results of their part, then the parts' maxima and sums.
constexpr size_t slab_floats(size_t head_dim) { return 16 * (head_dim + 2); }
constexpr size_t slabs_of(size_t head_dim) { return kAttnRoundFloats / slab_floats(head_dim); }

// The counts that a captured launch, whose grid is fixed, reads.
struct BatchHead {
    uint32_t n_seqs, n_tokens;
    uint32_t n_joins, join_rows;  // the most rows of a split tile
    uint32_t first[kClasses + 1];  // a class's items: [first[c], first[c + 1])
};
// A batch's arrays in device memory.
struct BatchView {
    const BatchHead *head;
    const SeqAt *seqs;
    const TokenAt *tokens;
    const uint32_t *pages;
    const uint64_t *tree;  // [token][kTreeWords]: which of its sequence's tokens it sees
    const ItemAt *items;
    const JoinAt *joins;
    int page_shift;
};

// The most blocks that a class's splits come to: four rounds of 512.
constexpr size_t kMostSplitBlocks = 2048;
// What a plan may hold, and what it is made for.
struct PlanShape {
    size_t n_kv_heads, head_dim, group, max_items, max_joins;
    bool bf16;
    unsigned classes;  // a bit for each class that may be used: the first always
    bool all_classes;  // each is, for the rows it is made for, whatever the estimate (tests)
};
// The most items and split tiles of a batch.
size_t most_items(size_t n_heads, size_t n_kv_heads, size_t max_seqs, size_t max_tokens);
size_t most_joins(size_t n_heads, size_t n_kv_heads, size_t max_seqs, size_t max_tokens);
// The classes that a captured call launches: those of the sequences' rows, which
// other lengths may want, those of the plan, and the first.
unsigned classes_of(const PlanShape &shape, const BatchHead &head, const SeqAt *seqs);
// Plans the attention of the head's sequences.
void plan_attention(const PlanShape &shape, const SeqAt *seqs, BatchHead *head, ItemAt *items, JoinAt *joins);

// q_out = q normalized and rotated; keys (normalized and rotated) and values to
// the cache. `n` tokens are launched for, those of the head are done.
struct PagedAppendArgs {
    BatchView b;
    float *q_out;
    const float *q, *k, *v;
    const uint16_t *q_norm, *k_norm;  // may be null
    const float *rope;
    void *cache;
    int n_heads, n_kv_heads;
    float eps;
};
hipError_t launch_paged_append(hipStream_t s, const PagedAppendArgs &a, size_t n, size_t head_dim, bool bf16);

struct PagedAttnArgs {
    BatchView b;
    float *out;
    const float *q;
    const void *cache;
    int n_heads, n_kv_heads, group;
    float scale;
    float *part;  // slabs
};
// `count`: what is set now, to be launched for. `captured`: not zero where what is
// set later is launched for too, by these classes.
hipError_t launch_paged_attention(hipStream_t s, const PagedAttnArgs &a, const BatchHead &count, size_t head_dim, bool bf16,
                                  unsigned captured);

// How many of `n` rows one launch of the argmax takes, in how many parts a row:
// [i * part, (i + 1) * part), the last to the row's end, so that none is empty.
// About 2048 blocks, of 4096 values at least; `rows * splits` results at most
// kMostPicks.
constexpr size_t kMostPicks = kPinnedFloats / 2;
struct RowParts {
    size_t rows, splits, part;
};
inline RowParts row_parts(size_t n, size_t cols) {
    const size_t rows = std::min(n, kMostPicks);
    const size_t most = std::max<size_t>(1, std::min({(cols + 4095) / 4096, (2048 + rows - 1) / rows, kMostPicks / rows}));
    const size_t part = ((cols + most - 1) / most + 3) / 4 * 4;
    return {rows, (cols + part - 1) / part, part};
}
// picks[row * splits + split] = the packed argmax of a part of a row.
hipError_t launch_argmax_rows(hipStream_t s, const float *x, size_t rows, size_t cols, const RowParts &parts, uint64_t *picks);

// Rows to move in every layer's cache, as kernel arguments: of segment i (a
// sequence) moves [start[i], start[i + 1]), in order.
struct PagedMove {
    uint32_t from, to;
};
constexpr int kMoves = 256, kMoveSegments = 64, kMoveLayers = 64;
struct PagedMoves {
    int n_segments, n_layers;
    int page_shift, n_kv_heads, row_bytes;  // row_bytes: of one head's row
    uint32_t start[kMoveSegments + 1];
    PagedMove move[kMoves];
    void *cache[kMoveLayers];
};
static_assert(sizeof(PagedMoves) <= 4096, "kernel arguments");
hipError_t launch_paged_moves(hipStream_t s, const PagedMoves &m);

// What the calls of one capture, or of the graph that it became, can take.
struct Captured {
    uint64_t capture;
    size_t tokens, positions;
    unsigned classes;
};

// Copies of up to eight arrays from pinned host memory in one launch (16-byte
// units; the addresses are multiples of 16).
struct Upload {
    const void *from[8];
    void *to[8];
    uint32_t units[8];
};
hipError_t launch_upload(hipStream_t s, const Upload &u);

}  // namespace th

// A step's sequences. The arrays exist twice: in pinned host memory, where
// th_batch_set writes them, and on the device, where one launch copies what is
// in use. Their places never change, so that a captured call reads what was
// set last.
struct th_batch {
    // What its caches are.
    size_t pages = 0, page_len = 0, n_kv_heads = 0, head_dim = 0;
    int kv_dtype = TH_KV_F32;
    th_device *dev = nullptr;  // whose stream it is copied on
    int page_shift = 0;
    size_t n_heads = 0, max_seqs = 0, max_tokens = 0, max_pages = 0;
    // Of what is set: sequences, tokens, entries of pages, the positions that a
    // rotation's table holds at least.
    size_t n_seqs = 0, n_tokens = 0, n_pages = 0, positions = 0;
    // The fewest tokens that a captured call was launched for, and the fewest
    // positions that a rotation's table of one holds.
    size_t captured_tokens = SIZE_MAX, captured_positions = SIZE_MAX;
    // The classes of the attention's items that every captured call launches, of
    // those that there are.
    unsigned classes = (1u << th::kClasses) - 1, all = classes;
    // The captures whose graphs there are, or that are open, and the least of each.
    th::Captured *captures = nullptr;
    size_t n_captures = 0, captures_room = 0;
    th_batch *next = nullptr;  // of the device's
    bool all_classes = false;
    char *device = nullptr, *pinned = nullptr;
    // Offsets, the same in both.
    size_t at_seqs = 0, at_tokens = 0, at_pages = 0, at_tree = 0, at_items = 0, at_joins = 0;
    hipEvent_t copied = nullptr;  // the pinned memory has been read
    int32_t *parents = nullptr;   // [max_tokens], -1: the context
    uint32_t *stamp = nullptr;    // [pages]: the last set() that wrote to a page
    uint32_t epoch = 0;

    th::BatchHead *head() const { return reinterpret_cast<th::BatchHead *>(pinned); }
    th::SeqAt *seqs() const { return reinterpret_cast<th::SeqAt *>(pinned + at_seqs); }
    uint32_t *page_list() const { return reinterpret_cast<uint32_t *>(pinned + at_pages); }
    th::PlanShape plan_shape() const {
        return {n_kv_heads, head_dim, n_heads / n_kv_heads, th::most_items(n_heads, n_kv_heads, max_seqs, max_tokens),
                th::most_joins(n_heads, n_kv_heads, max_seqs, max_tokens), kv_dtype == TH_KV_BF16, classes, all_classes};
    }
    th::BatchView view() const {
        return {reinterpret_cast<const th::BatchHead *>(device),
                reinterpret_cast<const th::SeqAt *>(device + at_seqs),
                reinterpret_cast<const th::TokenAt *>(device + at_tokens),
                reinterpret_cast<const uint32_t *>(device + at_pages),
                reinterpret_cast<const uint64_t *>(device + at_tree),
                reinterpret_cast<const th::ItemAt *>(device + at_items),
                reinterpret_cast<const th::JoinAt *>(device + at_joins),
                page_shift};
    }
};

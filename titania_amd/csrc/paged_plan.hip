// The plan of a step's attention over a paged cache (host code): tiles of rows,
// and their positions split so that the launch fills the chip.
#include <algorithm>

#include "paged.h"

namespace th {

namespace {

// Blocks that a step is split for, where its positions allow: two of four
// waves a CU.
constexpr size_t kBlocks = 512;
// A block's fewest positions: one step of its four waves.
constexpr size_t kStep = 64;

}  // namespace

size_t most_joins(size_t n_heads, size_t n_kv_heads, size_t max_seqs, size_t max_tokens) {
    return max_tokens * (n_heads / n_kv_heads) / kClassRows[0] + max_seqs;
}

size_t most_items(size_t n_heads, size_t n_kv_heads, size_t max_seqs, size_t max_tokens) {
    return most_joins(n_heads, n_kv_heads, max_seqs, max_tokens) + kBlocks;
}

void plan_attention(const PlanShape &shape, const SeqAt *seqs, BatchHead *head, ItemAt *items, JoinAt *joins) {
    // A tile takes the smallest class that holds what is left of its sequence,
    // or the largest there is.
    auto class_of = [&](size_t rows) {
        int best = 0;
        for (int c = 0; c < kClasses; ++c)
            if (shape.classes >> c & 1 && (shape.head_dim < 256 || c == 0)) {
                best = c;
                if (rows <= (size_t)kClassRows[c]) break;
            }
        return best;
    };
    // f(class, sequence, first row, positions) for each tile.
    auto each_tile = [&](auto f) {
        for (uint32_t s = 0; s < head->n_seqs; ++s) {
            const size_t rows = seqs[s].n_new * shape.group;
            for (size_t r = 0; r < rows;) {
                const int c = class_of(rows - r);
                const size_t end = std::min(rows, r + kClassRows[c]);
                f(c, s, (uint32_t)r, (size_t)seqs[s].context + (end - 1) / shape.group + 1);
                r = end;
            }
        }
    };
    size_t steps = 0;
    each_tile([&](int, uint32_t, uint32_t, size_t len) { steps += (len + kStep - 1) / kStep; });
    const size_t target = std::max<size_t>(1, kBlocks / shape.n_kv_heads);
    const size_t most = std::max<size_t>(1, (steps + target - 1) / target);  // steps of an item
    uint32_t n_items = 0, part = 0;
    const uint32_t parts = (uint32_t)slabs_of(shape.head_dim);
    head->n_joins = head->join_rows = 0;
    for (int c = 0; c < kClasses; ++c) {
        head->first[c] = n_items;
        each_tile([&](int of, uint32_t s, uint32_t row0, size_t len) {
            if (of != c) return;
            const size_t n = (len + kStep - 1) / kStep;
            size_t splits = (n + most - 1) / most;
            const uint32_t slabs = kClassRows[c] / 16, each = slabs * (uint32_t)shape.n_kv_heads;
            if (splits * each > parts - part || head->n_joins == shape.max_joins) splits = 1;
            if (splits > 1) {
                joins[head->n_joins++] = {s, row0, part, (uint32_t)splits, slabs};
                head->join_rows = std::max(head->join_rows, std::min<uint32_t>(kClassRows[c], seqs[s].n_new * shape.group - row0));
            }
            for (size_t i = 0; i < splits; ++i) {
                const size_t k0 = i * n / splits * kStep, k1 = std::min(len, (i + 1) * n / splits * kStep);
                items[n_items++] = {s, row0, (uint32_t)k0, (uint32_t)k1, splits > 1 ? part : kNoPart};
                if (splits > 1) part += each;
            }
        });
    }
    head->first[kClasses] = n_items;
}

}  // namespace th

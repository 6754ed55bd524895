// The plan of a step's attention over a paged cache (host code): tiles of rows,
// and their positions split so that the launch fills the chip.
#include <algorithm>

#include "paged.h"

namespace th {

namespace {

// What the chip holds of a class's blocks at once: two a CU, or one where LDS
// or registers hold no more. (Trees of 14 to 25 tokens over bf16, whose class 1
// fits twice in 128 registers a thread, 50 -> 43 us.) These numbers and the
// estimates below are of head_dim 128, and 64 and 256 take them as they are: 64
// tokens at 120 to 8000 still run at 5.6 (f32) and 4.8 TB/s (bf16) of keys and
// values with heads of 64, 5.8 and 4.6 with 256, where 128 has 5.8 and 5.2.
constexpr size_t kSlots[kClasses] = {512, 256, 256}, kSlotsBf16[kClasses] = {512, 512, 256};
// An estimate of a block's time in us: for each 64 positions, alone and with the
// chip full of others, and for the rest of it and its launch; fitted to measured
// calls. (Splits into one round, whatever the lengths, 64 tokens at 120 to 8000
// 228 -> 209 us, those trees 61 -> 50.)
constexpr double kAloneUs[kClasses] = {1.5, 2.8, 4.5}, kAloneUsBf16[kClasses] = {1.5, 2.5, 3.5};
constexpr double kFullUs[kClasses] = {5.7, 3.7, 6.0}, kFullUsBf16[kClasses] = {3.2, 4.1, 3.7};
constexpr double kBlockUs[kClasses] = {5.0, 8.0, 10.0};
// Of the second launch that joins split tiles, by their class, and the bytes of
// partial results that are written, or read, in a microsecond.
constexpr double kJoinUs[kClasses] = {2.5, 6.5, 6.5}, kBytesUs = 6e6;
// The most rounds of blocks that a class is split into.
constexpr size_t kRounds = 4;
static_assert(kRounds * kSlotsBf16[0] <= kMostSplitBlocks && kRounds * kSlotsBf16[1] <= kMostSplitBlocks, "splits");
// A block's fewest positions: one step of its waves.
constexpr size_t kStep = 64;

// A sequence takes the smallest class that holds its rows, or the largest there
// is, with all of its tiles: a few rows that are left over run beside the others.
int class_of(const PlanShape &shape, size_t rows, unsigned classes) {
    int best = 0;
    for (int c = 0; c < kClasses; ++c)
        if (classes >> c & 1 && (shape.head_dim < 256 || c == 0)) {
            best = c;
            if (rows <= (size_t)kClassRows[c]) break;
        }
    return best;
}

}  // namespace

unsigned classes_of(const PlanShape &shape, const BatchHead &head, const SeqAt *seqs) {
    unsigned classes = 1;
    for (uint32_t s = 0; s < head.n_seqs; ++s) classes |= 1u << class_of(shape, seqs[s].n_new * shape.group, shape.classes);
    for (int c = 0; c < kClasses; ++c) classes |= (unsigned)(head.first[c + 1] > head.first[c]) << c;
    return classes;
}

size_t most_joins(size_t n_heads, size_t n_kv_heads, size_t max_seqs, size_t max_tokens) {
    return max_tokens * (n_heads / n_kv_heads) / kClassRows[0] + max_seqs;
}

size_t most_items(size_t n_heads, size_t n_kv_heads, size_t max_seqs, size_t max_tokens) {
    return most_joins(n_heads, n_kv_heads, max_seqs, max_tokens) + kClasses * kMostSplitBlocks;
}

void plan_attention(const PlanShape &shape, const SeqAt *seqs, BatchHead *head, ItemAt *items, JoinAt *joins) {
    // f(sequence, first row, positions) for each tile of a class, in order.
    auto each_tile = [&](int c, unsigned classes, auto f) {
        for (uint32_t s = 0; s < head->n_seqs; ++s) {
            const size_t rows = seqs[s].n_new * shape.group;
            if (rows == 0 || class_of(shape, rows, classes) != c) continue;
            for (size_t r = 0; r < rows; r += kClassRows[c]) {
                const size_t end = std::min(rows, r + kClassRows[c]);
                f(s, (uint32_t)r, (size_t)seqs[s].context + (end - 1) / shape.group + 1);
            }
        }
    };
    // The most steps of a class's items, and an estimate of its time without the
    // join: as they are, in ceil(blocks / slots) rounds or what the longest first
    // leaves of them, or such that the blocks fill 1 to kRounds rounds.
    struct Cut {
        size_t most;
        double us;
        bool split;
    };
    auto cut_of = [&](int c, unsigned classes) {
        size_t steps = 0, tiles = 0, longest = 0;
        each_tile(c, classes, [&](uint32_t, uint32_t, size_t len) {
            const size_t n = (len + kStep - 1) / kStep;
            steps += n;
            ++tiles;
            longest = std::max(longest, n);
        });
        if (!tiles) return Cut{0, 0, false};
        auto items_at = [&](size_t most) {
            size_t items = 0;
            each_tile(c, classes, [&](uint32_t, uint32_t, size_t len) { items += ((len + kStep - 1) / kStep + most - 1) / most; });
            return items;
        };
        // Partial results, written and read once.
        auto parts_us = [&](size_t most) {
            size_t rows = 0;
            each_tile(c, classes, [&](uint32_t s, uint32_t row0, size_t len) {
                const size_t splits = ((len + kStep - 1) / kStep + most - 1) / most;
                if (splits > 1) rows += splits * std::min<size_t>(kClassRows[c], seqs[s].n_new * shape.group - row0);
            });
            return (double)(rows * shape.n_kv_heads * (shape.head_dim + 2)) * 8 / kBytesUs;
        };
        const double slots = (double)(shape.bf16 ? kSlotsBf16 : kSlots)[c] / shape.n_kv_heads;  // of items
        const double alone = (shape.bf16 ? kAloneUsBf16 : kAloneUs)[c], full = (shape.bf16 ? kFullUsBf16 : kFullUs)[c];
        auto step_us = [&](double items) { return alone + (full - alone) * std::min(1.0, items / slots); };
        Cut best{longest, std::max(longest * step_us(tiles), steps / slots * full) + std::max(1.0, tiles / slots) * kBlockUs[c],
                 false};
        for (size_t r = 1; r <= kRounds; ++r) {
            const size_t room = std::max<size_t>(1, (size_t)(r * slots));
            if (room <= tiles) continue;
            size_t low = std::max<size_t>(1, (steps + room - 1) / room), high = longest;
            while (low < high) {
                const size_t mid = (low + high) / 2;
                if (items_at(mid) <= room) high = mid;
                else low = mid + 1;
            }
            if (low == longest) continue;
            const double us = r * (low * step_us((double)items_at(low) / r) + kBlockUs[c]) + parts_us(low);
            if (us + kJoinUs[c] < best.us + (best.split ? kJoinUs[c] : 0)) best = {low, us, true};
        }
        return best;
    };
    // Each class is a launch, and the launches run one after another; large tiles
    // have more partial results and a longer start, small ones read keys and values
    // more often. So fewer classes where that is less, by an estimate that is off
    // by up to a twentieth. Of the first 260 attentions that
    // perf/more_operators.py draws with random.Random(5), 78 are cut differently
    // so, and take 13.1 us where they took 18.2 (geometric means; at worst 1.07
    // times as long, at best 0.28: profiles/paged_plan.md). f32, 32 / 8 heads, with
    // the smallest class for each and now: 16 trees of up to 6 tokens at 800
    // 38 -> 32, 24 chunks of up to 38 at 30 28 -> 13, a tree of 60 at 300 23 -> 18, at
    // 3900 38 -> 33, and from 8100 on as it was.
    Cut cuts[kClasses] = {};
    unsigned classes = 0;
    double least = 0;
    for (unsigned now : {7u, 3u, 1u}) {
        now &= shape.classes;
        bool other = !classes;  // than what there is: without a class that has tiles
        for (int c = 0; c < kClasses; ++c) other = other || ((classes & ~now) >> c & 1 && cuts[c].most);
        if (!other) continue;
        Cut mine[kClasses];
        double us = 0, join = 0;
        for (int c = 0; c < kClasses; ++c) {
            mine[c] = cut_of(c, now);
            us += mine[c].us;
            if (mine[c].split) join = std::max(join, kJoinUs[c]);
        }
        us += join;
        if (!classes || us < 0.95 * least) {
            std::copy(mine, mine + kClasses, cuts);
            classes = now;
            least = us;
        }
        if (shape.all_classes) break;
    }
    uint32_t n_items = 0, part = 0;
    const uint32_t parts = (uint32_t)slabs_of(shape.head_dim);
    head->n_joins = head->join_rows = 0;
    for (int c = 0; c < kClasses; ++c) {
        head->first[c] = n_items;
        const size_t most = cuts[c].most;
        if (!most) continue;
        each_tile(c, classes, [&](uint32_t s, uint32_t row0, size_t len) {
            const size_t n = (len + kStep - 1) / kStep;
            size_t splits = (n + most - 1) / most;
            const uint32_t slabs = kClassRows[c] / 16, each = slabs * (uint32_t)shape.n_kv_heads;
            if (splits * each > parts - part || head->n_joins == shape.max_joins) splits = 1;
            if (splits > 1) {
                const uint32_t rows = std::min<uint32_t>(kClassRows[c], seqs[s].n_new * shape.group - row0);
                joins[head->n_joins++] = {seqs[s].token0, rows, row0, part, (uint32_t)splits, slabs};
                head->join_rows = std::max(head->join_rows, rows);
            }
            for (size_t i = 0; i < splits; ++i) {
                const size_t k0 = i * n / splits * kStep, k1 = std::min(len, (i + 1) * n / splits * kStep);
                items[n_items++] = {seqs[s], row0, (uint32_t)k0, (uint32_t)k1, splits > 1 ? part : kNoPart};
                if (splits > 1) part += each;
            }
        });
        // The longest first: blocks start in order, and short ones fill the end.
        std::sort(items + head->first[c], items + n_items, [](const ItemAt &x, const ItemAt &y) {
            const uint32_t m = x.k1 - x.k0, n = y.k1 - y.k0;
            return m != n ? m > n : x.seq.token0 != y.seq.token0 ? x.seq.token0 < y.seq.token0
                            : x.row0 != y.row0   ? x.row0 < y.row0
                                                 : x.k0 < y.k0;
        });
    }
    head->first[kClasses] = n_items;
}

}  // namespace th

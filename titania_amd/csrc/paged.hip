// The C ABI's paged caches (th_paged) and batches (th_batch): handles, host
// copies, argument checks, and what a step's calls read of its batch.
#include <algorithm>
#include <atomic>
#include <chrono>
#include <cstdlib>
#include <cstring>
#include <new>

#include "../../include/titania_hip_test_paged.h"
#include "paged.h"

using th::fail;

namespace {

// Handles of another GPU are refused.
#define TH_PAGED_HERE(dev, x) \
    TH_REQUIRE((x)->ordinal == (dev)->ordinal, "a handle of GPU %d on GPU %d", (x)->ordinal, (dev)->ordinal)
// A batch is copied on its device's stream, which no other one waits for.
#define TH_BATCH_OF(dev, b) TH_REQUIRE((b)->dev == (dev), "a batch belongs to the device it was allocated with")
#define TH_PAGED_CURRENT(dev)  \
    th::Current current_(dev); \
    TH_HIP(current_.error)

int hip_failed(hipError_t e, const char *what) {
    (void)hipGetLastError();  // reported here, not by the next launch
    return fail(e == hipErrorOutOfMemory ? TH_ERR_NOMEM : TH_ERR_HIP, "%s failed: %s", what, hipGetErrorString(e));
}

size_t row_bytes(const th_paged *c) { return c->head_dim * (c->kv_dtype == TH_KV_BF16 ? 2 : 4); }
size_t page_bytes(const th_paged *c) { return 2 * c->n_kv_heads * c->page_len * row_bytes(c); }

uint16_t to_bf16(float f) {
    uint32_t u;
    memcpy(&u, &f, 4);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)(u >> 16 | 0x40);
    return (uint16_t)((u + 0x7fff + (u >> 16 & 1)) >> 16);
}
float from_bf16(uint16_t b) {
    const uint32_t u = (uint32_t)b << 16;
    float f;
    memcpy(&f, &u, 4);
    return f;
}

// One page between the device and arrays [page_len][n_kv_heads][head_dim].
template <bool READ, typename F>
void reorder_page(const th_paged *c, char *raw, F *k, F *v) {
    for (size_t kv = 0; kv < 2; ++kv)
        for (size_t h = 0; h < c->n_kv_heads; ++h)
            for (size_t r = 0; r < c->page_len; ++r) {
                F *plain = (kv ? v : k) + (r * c->n_kv_heads + h) * c->head_dim;
                char *row = raw + ((kv * c->n_kv_heads + h) * c->page_len + r) * row_bytes(c);
                for (size_t i = 0; i < c->head_dim; ++i) {
                    auto *b = reinterpret_cast<uint16_t *>(row);
                    auto *f = reinterpret_cast<float *>(row);
                    if constexpr (READ) plain[i] = c->kv_dtype == TH_KV_BF16 ? from_bf16(b[i]) : f[i];
                    else if (c->kv_dtype == TH_KV_BF16) b[i] = to_bf16(plain[i]);
                    else f[i] = plain[i];
                }
            }
}

int same_cache(const th_device *dev, const th_paged *c, const th_batch *b) {
    TH_PAGED_HERE(dev, c);
    TH_BATCH_OF(dev, b);
    TH_REQUIRE(c->pages == b->pages && c->page_len == b->page_len && c->n_kv_heads == b->n_kv_heads &&
                   c->head_dim == b->head_dim && c->kv_dtype == b->kv_dtype,
               "a cache of %zu pages of %zu positions of %zu x %zu in type %d, a batch for %zu of %zu of %zu x %zu in type %d",
               c->pages, c->page_len, c->n_kv_heads, c->head_dim, c->kv_dtype, b->pages, b->page_len, b->n_kv_heads, b->head_dim,
               b->kv_dtype);
    return TH_OK;
}

// Whether a batch can be set to this. Changes nothing but the stamps.
int check_set(th_batch *b, size_t n_seqs, const uint32_t *context, const uint32_t *n_new, const uint32_t *pages, size_t n_pages,
              const int32_t *parents) {
    TH_REQUIRE(n_seqs == 0 || (context && n_new), "th_batch_set: null argument");
    TH_REQUIRE(n_pages == 0 || pages, "th_batch_set: null pages");
    TH_REQUIRE(n_seqs <= b->max_seqs, "%zu sequences, a batch of at most %zu", n_seqs, b->max_seqs);
    TH_REQUIRE(n_pages <= b->max_pages, "%zu pages, a batch of at most %zu", n_pages, b->max_pages);
    // Everything is checked before anything is changed.
    size_t tokens = 0, entries = 0;
    const size_t L = b->page_len;
    for (size_t s = 0; s < n_seqs; ++s) {
        const size_t len = (size_t)context[s] + n_new[s];
        entries += (len + L - 1) / L;
        tokens += n_new[s];
        TH_REQUIRE(entries <= n_pages, "sequence %zu of %zu positions is past the end of %zu pages", s, len, n_pages);
        TH_REQUIRE(tokens <= b->max_tokens, "%zu tokens up to sequence %zu, a batch of at most %zu", tokens, s, b->max_tokens);
        TH_REQUIRE(len <= th::kMostPositions, "%zu positions of sequence %zu: at most %zu", len, s, th::kMostPositions);
    }
    TH_REQUIRE(entries == n_pages, "%zu pages for sequences of %zu", n_pages, entries);
    TH_REQUIRE(tokens <= b->captured_tokens,
               "%zu tokens: a graph was captured with this batch at %zu, and its launches take no more", tokens,
               b->captured_tokens);
    for (size_t i = 0; i < n_pages; ++i)
        TH_REQUIRE(pages[i] < b->pages, "page %u at index %zu of a cache of %zu", pages[i], i, b->pages);
    // A page that gets new rows is in no other place of a sequence with tokens.
    if (++b->epoch == 0) {
        memset(b->stamp, 0, b->pages * sizeof(uint32_t));
        b->epoch = 1;
    }
    for (size_t s = 0, p0 = 0; s < n_seqs; ++s) {
        const size_t len = (size_t)context[s] + n_new[s], end = p0 + (len + L - 1) / L;
        for (size_t p = p0 + context[s] / L; n_new[s] && p < end; ++p) {
            TH_REQUIRE(b->stamp[pages[p]] != b->epoch, "page %u gets new rows in two places, one of them of sequence %zu",
                       pages[p], s);
            b->stamp[pages[p]] = b->epoch;
        }
        p0 = end;
    }
    for (size_t s = 0, p0 = 0; s < n_seqs; ++s) {
        const size_t len = (size_t)context[s] + n_new[s], end = p0 + (len + L - 1) / L;
        for (size_t p = p0; n_new[s] && p < p0 + context[s] / L; ++p)
            TH_REQUIRE(b->stamp[pages[p]] != b->epoch, "page %u gets new rows, and is in the context of sequence %zu", pages[p], s);
        p0 = end;
    }
    size_t positions = 0;  // that are rotated by
    for (size_t s = 0, t0 = 0; s < n_seqs; t0 += n_new[s++]) {
        bool chain = true;
        for (size_t i = 0; parents && i < n_new[s]; ++i) {
            TH_REQUIRE(parents[t0 + i] >= -1 && parents[t0 + i] < (int64_t)i, "parent %d of token %zu of sequence %zu",
                       parents[t0 + i], i, s);
            chain = chain && parents[t0 + i] == (int64_t)i - 1;
        }
        TH_REQUIRE(chain || n_new[s] <= th::kTreeTokens, "a tree of %u tokens: at most %zu", n_new[s], th::kTreeTokens);
        size_t deep = chain ? n_new[s] : 0, level[th::kTreeTokens];
        for (size_t i = 0; !chain && i < n_new[s]; ++i) {
            level[i] = parents[t0 + i] < 0 ? 1 : level[parents[t0 + i]] + 1;
            deep = std::max(deep, level[i]);
        }
        if (n_new[s]) positions = std::max(positions, context[s] + deep);
    }
    TH_REQUIRE(positions <= b->captured_positions,
               "position %zu: a graph was captured with this batch over a table of %zu, past whose end it would read",
               positions - 1, b->captured_positions);
    return TH_OK;
}

// Its arrays in pinned memory. Returns the tokens up to the end of the last tree.
size_t lay_out(th_batch *b, size_t n_seqs, const uint32_t *context, const uint32_t *n_new, const uint32_t *pages, size_t n_pages,
               const int32_t *parents) {
    const size_t L = b->page_len;
    size_t tokens = 0;
    for (size_t s = 0; s < n_seqs; ++s) tokens += n_new[s];
    auto *head = b->head();
    auto *seqs = b->seqs();
    auto *toks = reinterpret_cast<th::TokenAt *>(b->pinned + b->at_tokens);
    auto *tree = reinterpret_cast<uint64_t *>(b->pinned + b->at_tree);
    head->n_seqs = (uint32_t)n_seqs;
    head->n_tokens = (uint32_t)tokens;
    if (n_pages) memcpy(b->page_list(), pages, n_pages * sizeof(uint32_t));
    size_t positions = 0, t0 = 0, p0 = 0, trees = 0;
    for (size_t s = 0; s < n_seqs; ++s) {
        const uint32_t n = n_new[s], ctx = context[s];
        int32_t *par = b->parents + t0;
        bool chain = true;
        for (uint32_t i = 0; i < n; ++i) {
            par[i] = parents ? parents[t0 + i] : (int32_t)i - 1;
            chain = chain && par[i] == (int32_t)i - 1;
        }
        seqs[s] = {(uint32_t)t0, n, ctx, (uint32_t)p0, !chain};
        for (uint32_t i = 0; i < n; ++i) {
            const size_t at = (size_t)ctx + i;
            th::TokenAt &t = toks[t0 + i];
            t.slot = pages[p0 + at / L] << b->page_shift | (uint32_t)(at & (L - 1));
            t.pos = par[i] < 0 ? ctx : toks[t0 + par[i]].pos + 1;
            positions = std::max<size_t>(positions, (size_t)t.pos + 1);
            if (chain) continue;
            uint64_t *bits = tree + (t0 + i) * th::kTreeWords;
            for (int w = 0; w < th::kTreeWords; ++w) bits[w] = par[i] < 0 ? 0 : tree[(t0 + par[i]) * th::kTreeWords + w];
            bits[i / 64] |= (uint64_t)1 << (i & 63);
        }
        if (!chain) trees = t0 + n;
        t0 += n;
        p0 += ((size_t)ctx + n + L - 1) / L;
    }
    b->n_seqs = n_seqs;
    b->n_tokens = tokens;
    b->n_pages = n_pages;
    b->positions = positions;
    auto *items = reinterpret_cast<th::ItemAt *>(b->pinned + b->at_items);
    auto *joins = reinterpret_cast<th::JoinAt *>(b->pinned + b->at_joins);
    th::plan_attention(b->plan_shape(), seqs, head, items, joins);
    return trees;
}

// A batch's offsets, and its host memory but for the pinned. False: there is none.
bool place_arrays(th_batch *b, size_t *bytes) {
    size_t at = 64;
    auto place = [&at](size_t n) {
        const size_t here = at;
        at += (n + 63) / 64 * 64;
        return here;
    };
    b->page_shift = __builtin_ctzll(b->page_len);
    b->at_seqs = place(b->max_seqs * sizeof(th::SeqAt));
    b->at_tokens = place(b->max_tokens * sizeof(th::TokenAt));
    b->at_pages = place(b->max_pages * sizeof(uint32_t));
    b->at_tree = place(b->max_tokens * th::kTreeWords * sizeof(uint64_t));
    b->at_items = place(b->plan_shape().max_items * sizeof(th::ItemAt));
    b->at_joins = place(b->plan_shape().max_joins * sizeof(th::JoinAt));
    *bytes = at;
    b->parents = static_cast<int32_t *>(malloc(b->max_tokens * sizeof(int32_t)));
    b->stamp = static_cast<uint32_t *>(calloc(b->pages, sizeof(uint32_t)));
    return b->parents && b->stamp;
}

// After a set that the GPU failed: the host's arrays may be the new step's and
// the device's another's, so nothing is set any more.
int set_failed(th_batch *b, hipError_t e) {
    if (b->dev) (void)hipStreamSynchronize(b->dev->stream);  // (a copy that did start)
    b->n_seqs = b->n_tokens = b->n_pages = b->positions = 0;
    *b->head() = {};
    return hip_failed(e, "setting a batch");
}

// Whether n words that a launch writes to pinned memory have all become other
// than zero, waited for without the runtime for a short while: what it takes to
// see a stream's end is more than what small launches take (24 rows of 151936
// 17.9 -> 13.3 us). The stream's end tells of the others, and of errors.
bool arrive(const uint64_t *words, size_t n) {
    const volatile uint64_t *w = words;
    const auto until = std::chrono::steady_clock::now() + std::chrono::microseconds(200);
    for (size_t i = 0; i < n; ++i)
        while (!w[i]) {
            for (int k = 0; k < 64 && !w[i]; ++k) __builtin_ia32_pause();
            if (!w[i] && std::chrono::steady_clock::now() > until) return false;
        }
    std::atomic_thread_fence(std::memory_order_acquire);
    return true;
}

// What all captures of a batch can take.
void weigh_captures(th_batch *b) {
    b->captured_tokens = b->captured_positions = SIZE_MAX;
    b->classes = b->all;
    for (size_t i = 0; i < b->n_captures; ++i) {
        b->captured_tokens = std::min(b->captured_tokens, b->captures[i].tokens);
        b->captured_positions = std::min(b->captured_positions, b->captures[i].positions);
        b->classes &= b->captures[i].classes;
    }
}

// A captured call is launched for the tokens that are set now, an append reads
// the table it was given, an attention launches some classes: as long as there is
// a graph of it, later sets may have no more tokens, none that are rotated by
// a position past the table's end, and a plan of those classes.
int note_capture(const th_device *dev, const th_batch *batch, size_t positions, unsigned classes) {
    if (!dev->capturing) return TH_OK;
    auto *b = const_cast<th_batch *>(batch);
    b->dev->captured_batch = true;
    size_t i = 0;
    while (i < b->n_captures && b->captures[i].capture != dev->capture) ++i;
    if (i == b->n_captures) {
        if (i == b->captures_room) {
            const size_t room = std::max<size_t>(8, 2 * i);
            auto *more = static_cast<th::Captured *>(realloc(b->captures, room * sizeof(th::Captured)));
            if (!more) return fail(TH_ERR_NOMEM, "out of host memory");
            b->captures = more;
            b->captures_room = room;
        }
        b->captures[b->n_captures++] = {dev->capture, SIZE_MAX, SIZE_MAX, ~0u};
    }
    th::Captured &c = b->captures[i];
    c.tokens = std::min(c.tokens, b->n_tokens);
    c.positions = std::min(c.positions, positions);
    c.classes &= classes;
    weigh_captures(b);
    return TH_OK;
}

// A batch without a device, in plain host memory.
struct HostBatch : th_batch {
    explicit HostBatch(const size_t *shape) {
        pages = shape[0];
        page_len = shape[1];
        n_kv_heads = shape[2];
        head_dim = shape[3];
        kv_dtype = (int)shape[4];
        n_heads = shape[5];
        max_seqs = shape[6];
        max_tokens = shape[7];
        max_pages = shape[8];
        size_t bytes = 0;
        if (place_arrays(this, &bytes)) pinned = static_cast<char *>(calloc(1, bytes));
    }
    ~HostBatch() {
        free(pinned);
        free(parents);
        free(stamp);
    }
};

}  // namespace

namespace th {

void release_capture(th_device *dev, uint64_t capture) {
    for (th_batch *b = dev->batches; b; b = b->next)
        for (size_t i = 0; i < b->n_captures; ++i)
            if (b->captures[i].capture == capture) {
                b->captures[i] = b->captures[--b->n_captures];
                weigh_captures(b);
                break;
            }
}

void leave_batches(th_device *dev) {
    while (th_batch *b = dev->batches) {
        dev->batches = b->next;
        b->dev = nullptr;
        b->next = nullptr;
    }
}

}  // namespace th

extern "C" {

int th_paged_alloc(th_device *dev, size_t pages, size_t page_len, size_t n_kv_heads, size_t head_dim, int kv_dtype,
                   th_paged **out) {
    TH_REQUIRE(dev && out, "th_paged_alloc: null argument");
    TH_NOT_CAPTURING(dev, "th_paged_alloc");
    TH_REQUIRE(page_len >= 16 && page_len <= 256 && (page_len & (page_len - 1)) == 0,
               "pages of %zu positions: 16, 32, 64, 128 or 256", page_len);
    TH_REQUIRE(pages > 0 && pages <= 0x7fffffffu / page_len, "%zu pages of %zu positions: 1 to 2^31 - 1 positions", pages,
               page_len);
    TH_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "head_dim %zu is not 64, 128 or 256", head_dim);
    TH_REQUIRE(n_kv_heads > 0 && n_kv_heads <= 1024, "%zu KV heads: 1 to 1024", n_kv_heads);
    TH_REQUIRE(kv_dtype == TH_KV_F32 || kv_dtype == TH_KV_BF16, "kv_dtype %d", kv_dtype);
    TH_PAGED_CURRENT(dev);
    auto *c = new (std::nothrow) th_paged();
    if (!c) return fail(TH_ERR_NOMEM, "out of host memory");
    c->pages = pages;
    c->page_len = page_len;
    c->n_kv_heads = n_kv_heads;
    c->head_dim = head_dim;
    c->kv_dtype = kv_dtype;
    c->ordinal = dev->ordinal;
    const size_t bytes = pages * page_bytes(c);  // below 2^31 * 2 * 2^10 * 2^10
    hipError_t e = hipMalloc(&c->ptr, bytes);
    if (e == hipSuccess) e = hipMemsetAsync(c->ptr, 0, bytes, dev->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(dev->stream);
    if (e != hipSuccess) {
        if (c->ptr) (void)hipFree(c->ptr);
        delete c;
        return hip_failed(e, "the allocation of a paged cache");
    }
    *out = c;
    return TH_OK;
}

void th_paged_free(th_device *dev, th_paged *c) {
    if (!c) return;
    if (dev && dev->capturing) {  // the handle stays valid: free it after th_graph_end
        fail(TH_ERR_INVALID, "th_paged_free cannot run while the device's stream is being captured");
        return;
    }
    if (dev) (void)hipStreamSynchronize(dev->stream);
    if (c->ptr) (void)hipFree(c->ptr);
    delete c;
}

int th_paged_shape(const th_paged *c, size_t *pages, size_t *page_len, size_t *n_kv_heads, size_t *head_dim, int *kv_dtype) {
    TH_REQUIRE(c && pages && page_len && n_kv_heads && head_dim && kv_dtype, "th_paged_shape: null argument");
    *pages = c->pages;
    *page_len = c->page_len;
    *n_kv_heads = c->n_kv_heads;
    *head_dim = c->head_dim;
    *kv_dtype = c->kv_dtype;
    return TH_OK;
}

int th_paged_read(th_device *dev, const th_paged *c, size_t page, float *k, float *v) {
    TH_REQUIRE(dev && c && k && v, "th_paged_read: null argument");
    TH_NOT_CAPTURING(dev, "th_paged_read");
    TH_PAGED_HERE(dev, c);
    TH_REQUIRE(page < c->pages, "page %zu of %zu", page, c->pages);
    TH_PAGED_CURRENT(dev);
    const size_t bytes = page_bytes(c);
    auto *raw = static_cast<char *>(malloc(bytes));
    if (!raw) return fail(TH_ERR_NOMEM, "out of host memory");
    hipError_t e = hipMemcpyAsync(raw, static_cast<const char *>(c->ptr) + page * bytes, bytes, hipMemcpyDeviceToHost, dev->stream);
    const hipError_t done = hipStreamSynchronize(dev->stream);
    if (e == hipSuccess) e = done;
    if (e == hipSuccess) reorder_page<true>(c, raw, k, v);
    free(raw);
    return e == hipSuccess ? TH_OK : hip_failed(e, "reading a page");
}

int th_paged_write(th_device *dev, th_paged *c, size_t page, const float *k, const float *v) {
    TH_REQUIRE(dev && c && k && v, "th_paged_write: null argument");
    TH_NOT_CAPTURING(dev, "th_paged_write");
    TH_PAGED_HERE(dev, c);
    TH_REQUIRE(page < c->pages, "page %zu of %zu", page, c->pages);
    TH_PAGED_CURRENT(dev);
    const size_t bytes = page_bytes(c);
    auto *raw = static_cast<char *>(malloc(bytes));
    if (!raw) return fail(TH_ERR_NOMEM, "out of host memory");
    reorder_page<false>(c, raw, k, v);
    hipError_t e = hipMemcpyAsync(static_cast<char *>(c->ptr) + page * bytes, raw, bytes, hipMemcpyHostToDevice, dev->stream);
    const hipError_t done = hipStreamSynchronize(dev->stream);  // raw is read until then
    if (e == hipSuccess) e = done;
    free(raw);
    return e == hipSuccess ? TH_OK : hip_failed(e, "writing a page");
}

void th_batch_free(th_device *dev, th_batch *b) {
    if (!b) return;
    if (dev && dev->capturing) {  // the handle stays valid: free it after th_graph_end
        fail(TH_ERR_INVALID, "th_batch_free cannot run while the device's stream is being captured");
        return;
    }
    if (dev) (void)hipStreamSynchronize(dev->stream);
    if (b->device) (void)hipFree(b->device);
    if (b->pinned) (void)hipHostFree(b->pinned);
    if (b->copied) (void)hipEventDestroy(b->copied);
    for (th_batch **at = b->dev ? &b->dev->batches : nullptr; at && *at; at = &(*at)->next)
        if (*at == b) {
            *at = b->next;
            break;
        }
    free(b->captures);
    free(b->parents);
    free(b->stamp);
    delete b;
}

int th_batch_alloc(th_device *dev, const th_paged *c, size_t n_heads, size_t max_seqs, size_t max_tokens, size_t max_pages,
                   th_batch **out) {
    TH_REQUIRE(dev && c && out, "th_batch_alloc: null argument");
    TH_NOT_CAPTURING(dev, "th_batch_alloc");
    TH_PAGED_HERE(dev, c);
    TH_REQUIRE(n_heads > 0 && n_heads % c->n_kv_heads == 0, "%zu query heads do not split into groups over %zu KV heads",
               n_heads, c->n_kv_heads);
    TH_REQUIRE(n_heads / c->n_kv_heads <= th::kPagedMaxGroup, "at most %zu query heads per KV head are supported",
               th::kPagedMaxGroup);
    TH_REQUIRE(max_seqs > 0 && max_seqs <= 65536, "%zu sequences: 1 to 65536", max_seqs);
    TH_REQUIRE(max_tokens > 0 && max_tokens <= ((size_t)1 << 24) / n_heads, "%zu tokens of %zu heads: 1 to 2^24 heads in all",
               max_tokens, n_heads);
    TH_REQUIRE(max_pages > 0 && max_pages <= (size_t)1 << 26, "%zu pages of a batch: 1 to 2^26", max_pages);
    TH_PAGED_CURRENT(dev);
    auto *b = new (std::nothrow) th_batch();
    if (!b) return fail(TH_ERR_NOMEM, "out of host memory");
    b->pages = c->pages;
    b->page_len = c->page_len;
    b->n_kv_heads = c->n_kv_heads;
    b->head_dim = c->head_dim;
    b->kv_dtype = c->kv_dtype;
    b->dev = dev;
    b->n_heads = n_heads;
    b->max_seqs = max_seqs;
    b->max_tokens = max_tokens;
    b->max_pages = max_pages;
    size_t at = 0;
    if (!place_arrays(b, &at)) {
        th_batch_free(nullptr, b);
        return fail(TH_ERR_NOMEM, "out of host memory");
    }
    hipError_t e = hipMalloc(reinterpret_cast<void **>(&b->device), at);
    if (e == hipSuccess) e = hipHostMalloc(reinterpret_cast<void **>(&b->pinned), at, hipHostMallocDefault);
    if (e == hipSuccess) e = hipEventCreateWithFlags(&b->copied, hipEventDisableTiming);
    if (e == hipSuccess) e = hipMemsetAsync(b->device, 0, at, dev->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(dev->stream);
    if (e != hipSuccess) {
        th_batch_free(nullptr, b);
        return hip_failed(e, "the allocation of a batch");
    }
    memset(b->pinned, 0, at);
    b->next = dev->batches;
    dev->batches = b;
    *out = b;
    return TH_OK;
}

int th_batch_set(th_device *dev, th_batch *b, size_t n_seqs, const uint32_t *context, const uint32_t *n_new,
                 const uint32_t *pages, size_t n_pages, const int32_t *parents) {
    TH_REQUIRE(dev && b, "th_batch_set: null argument");
    TH_NOT_CAPTURING(dev, "th_batch_set");
    TH_BATCH_OF(dev, b);
    TRY(check_set(b, n_seqs, context, n_new, pages, n_pages, parents));
    th::Current current(dev);
    hipError_t e = current.error;
    if (e == hipSuccess) e = hipEventSynchronize(b->copied);  // the copy before has read the pinned memory
    if (e != hipSuccess) return set_failed(b, e);
    const size_t trees = lay_out(b, n_seqs, context, n_new, pages, n_pages, parents);
    const th::BatchHead *head = b->head();
    th::Upload u{};
    int k = 0;
    auto add = [&](size_t at, size_t bytes) {
        u.from[k] = b->pinned + at;
        u.to[k] = b->device + at;
        u.units[k++] = (uint32_t)((bytes + 15) / 16);
    };
    add(0, sizeof(th::BatchHead));
    add(b->at_seqs, n_seqs * sizeof(th::SeqAt));
    add(b->at_tokens, b->n_tokens * sizeof(th::TokenAt));
    add(b->at_pages, n_pages * sizeof(uint32_t));
    add(b->at_tree, trees * th::kTreeWords * sizeof(uint64_t));
    add(b->at_items, head->first[th::kClasses] * sizeof(th::ItemAt));
    add(b->at_joins, head->n_joins * sizeof(th::JoinAt));
    e = th::launch_upload(dev->stream, u);
    if (e == hipSuccess) e = hipEventRecord(b->copied, dev->stream);
    return e == hipSuccess ? TH_OK : set_failed(b, e);
}

int th_paged_append(th_device *dev, th_buffer *q_out, const th_buffer *q, const th_buffer *k, const th_buffer *v,
                    const th_weight *q_norm, const th_weight *k_norm, const th_buffer *rope, th_paged *c, const th_batch *b,
                    float eps) {
    TH_REQUIRE(dev && q_out && q && k && v && rope && c && b, "th_paged_append: null argument");
    TRY(same_cache(dev, c, b));
    const size_t n = b->n_tokens, hd = b->head_dim;
    TH_REQUIRE(q->len == n * b->n_heads * hd && q_out->len == q->len,
               "q and q_out hold %zu and %zu activations, not %zu tokens of %zu x %zu", q->len, q_out->len, n, b->n_heads, hd);
    TH_REQUIRE(k->len == n * b->n_kv_heads * hd && v->len == k->len,
               "k and v hold %zu and %zu activations, not %zu tokens of %zu x %zu", k->len, v->len, n, b->n_kv_heads, hd);
    TH_REQUIRE(n == 0 || (q_out->ptr != k->ptr && q_out->ptr != v->ptr && q_out->ptr != rope->ptr),
               "q_out may be q, not k, v or the table");
    TH_REQUIRE((!q_norm || q_norm->numel == hd) && (!k_norm || k_norm->numel == hd), "q/k norms hold head_dim gains");
    TH_REQUIRE(b->positions * hd <= rope->len, "position %zu is past the end of the table", b->positions - 1);
    TH_PAGED_CURRENT(dev);
    th::PagedAppendArgs a{b->view(), q_out->ptr, q->ptr, k->ptr, v->ptr, q_norm ? q_norm->ptr : nullptr,
                          k_norm ? k_norm->ptr : nullptr, rope->ptr, c->ptr, (int)b->n_heads, (int)b->n_kv_heads, eps};
    TRY(note_capture(dev, b, rope->len / hd, ~0u));
    TH_HIP(th::launch_paged_append(dev->stream, a, n, hd, c->kv_dtype == TH_KV_BF16));
    return TH_OK;
}

int th_paged_attention(th_device *dev, th_buffer *out, const th_buffer *q, const th_paged *c, const th_batch *b) {
    TH_REQUIRE(dev && out && q && c && b, "th_paged_attention: null argument");
    TRY(same_cache(dev, c, b));
    const size_t n = b->n_tokens, hd = b->head_dim;
    TH_REQUIRE(q->len == n * b->n_heads * hd && out->len == q->len,
               "q and out hold %zu and %zu activations, not %zu tokens of %zu x %zu", q->len, out->len, n, b->n_heads, hd);
    TH_REQUIRE(n == 0 || out->ptr != q->ptr, "attention cannot write its queries");
    TH_PAGED_CURRENT(dev);
    th::PagedAttnArgs a{b->view(), out->ptr, q->ptr, c->ptr, (int)b->n_heads, (int)b->n_kv_heads,
                        (int)(b->n_heads / b->n_kv_heads), 1.0f / sqrtf((float)hd), dev->part};
    const unsigned captured = dev->capturing ? th::classes_of(b->plan_shape(), *b->head(), b->seqs()) : 0;
    TRY(note_capture(dev, b, SIZE_MAX, captured));
    TH_HIP(th::launch_paged_attention(dev->stream, a, *b->head(), hd, c->kv_dtype == TH_KV_BF16, captured));
    return TH_OK;
}

int th_batch_accept(th_device *dev, const th_batch *b, const th_buffer *logits, const uint32_t *tokens, uint32_t *picks,
                    uint32_t *n_kept, int32_t *kept) {
    TH_REQUIRE(dev && b && logits, "th_batch_accept: null argument");
    TH_NOT_CAPTURING(dev, "th_batch_accept");
    TH_BATCH_OF(dev, b);
    TH_REQUIRE(b->n_seqs == 0 || n_kept, "th_batch_accept: null output");
    const size_t n = b->n_tokens;
    if (n) {
        TH_REQUIRE(tokens && picks && kept, "th_batch_accept: null argument");
        TH_REQUIRE(logits->len > 0 && logits->len % n == 0, "%zu logits are not whole rows of %zu tokens", logits->len, n);
        const size_t vocab = logits->len / n;
        TH_REQUIRE(vocab < 0xffffffffu, "rows of %zu logits", vocab);
        TH_PAGED_CURRENT(dev);
        // Each block leaves its part's maximum in pinned memory; the host
        // takes the largest.
        auto *picked = reinterpret_cast<uint64_t *>(dev->pinned);
        const th::RowParts parts = th::row_parts(n, vocab);
        const size_t splits = parts.splits;
        for (size_t r = 0; r < n; r += parts.rows) {
            const size_t now = std::min(parts.rows, n - r);
            memset(picked, 0, now * splits * sizeof(uint64_t));  // no part's maximum: an index is below 2^32 - 1
            TH_HIP(th::launch_argmax_rows(dev->stream, logits->ptr + r * vocab, now, vocab, parts, picked));
            if (!arrive(picked, now * splits)) TH_HIP(hipStreamSynchronize(dev->stream));
            for (size_t i = 0; i < now; ++i) {
                const uint64_t best = *std::max_element(picked + i * splits, picked + (i + 1) * splits);
                picks[r + i] = 0xffffffffu - (uint32_t)best;
            }
        }
    }
    // From token 0 on, to the first child that is what its parent picked.
    const th::SeqAt *seqs = b->seqs();
    for (size_t s = 0; s < b->n_seqs; ++s) {
        const size_t t0 = seqs[s].token0, m = seqs[s].n_new;
        size_t k = 0;
        int32_t last = 0;
        if (m) kept[t0 + k++] = 0;
        for (size_t i = 1; i < m; ++i)  // a child comes after its parent
            if (b->parents[t0 + i] == last && tokens[t0 + i] == picks[t0 + last]) kept[t0 + k++] = last = (int32_t)i;
        n_kept[s] = (uint32_t)k;
        for (; k < m; ++k) kept[t0 + k] = -1;
    }
    return TH_OK;
}

int th_paged_keep(th_device *dev, th_paged *const *caches, size_t n_caches, const th_batch *b, const uint32_t *n_kept,
                  const int32_t *kept) {
    TH_REQUIRE(dev && b && (n_caches == 0 || caches), "th_paged_keep: null argument");
    TH_NOT_CAPTURING(dev, "th_paged_keep");
    TH_BATCH_OF(dev, b);
    for (size_t i = 0; i < n_caches; ++i) {
        TH_REQUIRE(caches[i], "th_paged_keep: null cache");
        TRY(same_cache(dev, caches[i], b));
        for (size_t j = 0; j < i; ++j) TH_REQUIRE(caches[i] != caches[j], "the same cache twice");
    }
    TH_REQUIRE(b->n_seqs == 0 || n_kept, "th_paged_keep: null argument");
    const th::SeqAt *seqs = b->seqs();
    for (size_t s = 0; s < b->n_seqs; ++s) {
        TH_REQUIRE(n_kept[s] <= seqs[s].n_new, "%u of %u tokens of sequence %zu kept", n_kept[s], seqs[s].n_new, s);
        TH_REQUIRE(n_kept[s] == 0 || kept, "th_paged_keep: null argument");
        for (uint32_t j = 0; j < n_kept[s]; ++j) {
            const int64_t at = kept[seqs[s].token0 + j], before = j ? kept[seqs[s].token0 + j - 1] : -1;
            TH_REQUIRE(at > before && at < seqs[s].n_new, "token %ld kept as number %u of sequence %zu, after token %ld", (long)at,
                       j, s, (long)before);
        }
    }
    if (n_caches == 0) return TH_OK;
    TH_PAGED_CURRENT(dev);
    th::PagedMoves m;
    m.page_shift = b->page_shift;
    m.n_kv_heads = (int)b->n_kv_heads;
    m.row_bytes = (int)row_bytes(caches[0]);
    m.n_segments = 0;
    uint32_t count = 0;
    auto flush = [&]() -> hipError_t {
        for (size_t c = 0; m.n_segments && c < n_caches; c += th::kMoveLayers) {
            m.n_layers = (int)std::min<size_t>(th::kMoveLayers, n_caches - c);
            for (int i = 0; i < m.n_layers; ++i) m.cache[i] = caches[c + i]->ptr;
            if (hipError_t e = th::launch_paged_moves(dev->stream, m); e != hipSuccess) return e;
        }
        m.n_segments = 0;
        count = 0;
        return hipSuccess;
    };
    const uint32_t *pages = b->page_list();
    for (size_t s = 0; s < b->n_seqs; ++s) {
        const th::SeqAt &q = seqs[s];
        auto slot = [&](size_t pos) {
            return pages[q.page0 + (pos >> b->page_shift)] << b->page_shift | (uint32_t)(pos & (b->page_len - 1));
        };
        bool open = false;  // the sequence has a segment of this launch
        for (uint32_t j = 0; j < n_kept[s]; ++j) {
            const uint32_t at = (uint32_t)kept[q.token0 + j];
            if (at == j) continue;
            if (count == th::kMoves || (!open && m.n_segments == th::kMoveSegments)) {
                TH_HIP(flush());
                open = false;
            }
            if (!open) {
                m.start[m.n_segments++] = count;
                open = true;
            }
            m.move[count++] = {slot((size_t)q.context + at), slot((size_t)q.context + j)};
            m.start[m.n_segments] = count;
        }
    }
    TH_HIP(flush());
    return TH_OK;
}

int th_test_accept_parts(size_t rows, size_t cols, size_t *rows_at_once, size_t *splits, size_t *part) {
    const th::RowParts parts = th::row_parts(rows, cols);
    *rows_at_once = parts.rows;
    *splits = parts.splits;
    *part = parts.part;
    return TH_OK;
}

int th_test_batch_classes(th_batch *b, unsigned classes) {
    TH_REQUIRE(b && classes < 1u << th::kClasses && classes & 1, "th_test_batch_classes: %u", classes);
    b->all = classes;
    b->all_classes = true;
    weigh_captures(b);
    return TH_OK;
}

int th_test_batch_set(const size_t *shape, unsigned classes, size_t captured_tokens, size_t captured_positions, size_t n_seqs,
                      const uint32_t *context, const uint32_t *n_new, const uint32_t *pages, size_t n_pages,
                      const int32_t *parents, uint32_t *tokens, uint64_t *tree, uint32_t *items, size_t *n_items,
                      uint32_t *joins, size_t *n_joins, uint32_t *first) {
    HostBatch b(shape);
    b.classes = classes;
    b.captured_tokens = captured_tokens;
    b.captured_positions = captured_positions;
    int rc = b.pinned ? check_set(&b, n_seqs, context, n_new, pages, n_pages, parents) : fail(TH_ERR_NOMEM, "out of host memory");
    if (rc == TH_OK) {
        lay_out(&b, n_seqs, context, n_new, pages, n_pages, parents);
        const th::BatchHead *head = b.head();
        const size_t most_items = *n_items, most_joins = *n_joins;
        *n_items = head->first[th::kClasses];
        *n_joins = head->n_joins;
        if (*n_items > std::min(most_items, b.plan_shape().max_items) || *n_joins > std::min(most_joins, b.plan_shape().max_joins)) {
            rc = fail(TH_ERR_INVALID, "%zu items and %zu joins", *n_items, *n_joins);
        } else {
            const auto *at = reinterpret_cast<const th::TokenAt *>(b.pinned + b.at_tokens);
            for (uint32_t s = 0; s < head->n_seqs; ++s)
                for (uint32_t i = 0; i < b.seqs()[s].n_new; ++i) {
                    const uint32_t t = b.seqs()[s].token0 + i;
                    const uint32_t now[] = {at[t].slot, at[t].pos, s, i};
                    memcpy(tokens + 4 * t, now, sizeof now);
                }
            memcpy(tree, b.pinned + b.at_tree, b.n_tokens * th::kTreeWords * sizeof(uint64_t));
            memcpy(items, b.pinned + b.at_items, *n_items * sizeof(th::ItemAt));
            memcpy(joins, b.pinned + b.at_joins, *n_joins * sizeof(th::JoinAt));
            memcpy(first, head->first, sizeof head->first);
        }
    }
    return rc;
}

int th_test_batch_set_failed(const size_t *shape, size_t n_seqs, const uint32_t *context, const uint32_t *n_new,
                             const uint32_t *pages, size_t n_pages, size_t *left) {
    HostBatch b(shape);
    if (!b.pinned) return fail(TH_ERR_NOMEM, "out of host memory");
    TRY(check_set(&b, n_seqs, context, n_new, pages, n_pages, nullptr));
    lay_out(&b, n_seqs, context, n_new, pages, n_pages, nullptr);
    const int rc = set_failed(&b, hipErrorLaunchFailure);
    const th::BatchHead *head = b.head();
    const size_t now[] = {b.n_seqs, b.n_tokens, b.n_pages, b.positions, head->n_seqs, head->n_tokens, head->n_joins,
                          head->join_rows, head->first[th::kClasses]};
    memcpy(left, now, sizeof now);
    return rc;
}

}  // extern "C"

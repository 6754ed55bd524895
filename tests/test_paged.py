"""Paged caches (th_paged) and the batches over them (th_batch): appends,
attention of ragged batches and drafted trees, verification, moved rows.

Results are compared with float64 under bounds for each element, with u = 2^-24
(half a step of f32):
- append: the norm's sum of head_dim squares, a division, a root and three
  products, then two products and a sum, (head_dim + 16) u of the pair's length;
  a bf16 cache rounds once more, half a step of which is 2^-8 of the value;
- attention: a score is off by the sum of head_dim products, by what the matrix
  cores' terms leave out (2^-21 of each product) and by the scale and the
  exponential (4 u of the score): d in all. Numerator and denominator of the
  softmax are each off by d and the sum over the keys, (keys + 8) u and 2^-21 of
  the weights' terms, so the result by twice that of sum p |v|.
"""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from titania_amd import TH_KV_BF16, TH_KV_F32, Hip, InvalidArgument, Tensor
from titania_amd._lib import LIB_PATH
from titania_amd._lib import check as ok
from titania_amd.synth import bf16_to_f32, f32_to_bf16

EPS = 1e-6
U = 2.0**-24
gpu = pytest.mark.gpu


def chain(n):
    return [i - 1 for i in range(n)]


def some_tree(r, n, back=6, roots=False):
    return [-1 if i == 0 or (roots and r.random() < 0.1) else int(r.integers(max(0, i - back), i)) for i in range(n)]


@pytest.fixture(params=[0, 7, 5])
def kernels(request):
    """Of the attention: those that the plan takes; each for the rows that it is
    made for; the one for up to 256 rows where the plan takes that for 128."""
    return request.param


def take(batch, kernels):
    if kernels:
        f = C.CDLL(str(LIB_PATH)).th_test_batch_classes
        f.argtypes = [C.c_void_p, C.c_uint]
        ok(f(batch.handle, kernels))


class Step:
    """Sequences with their pages in random order, and what each token sees."""

    def __init__(self, r, context, new, page_len, trees=None, spare=3, shared=0):
        self.context, self.new, self.L = list(context), list(new), page_len
        self.first = [sum(new[:s]) for s in range(len(new))]
        self.tokens = sum(new)
        need = [-(-(c + n) // page_len) for c, n in zip(context, new)]
        self.pages = sum(need) + spare
        ids = list(r.permutation(self.pages))
        # The first `shared` pages of every context are sequence 0's.
        self.lists = []
        for s, (n, c) in enumerate(zip(need, context)):
            got = [ids.pop() for _ in range(n)]
            for i in range(min(shared, c // page_len, len(self.lists[0]) if s else 0)):
                got[i] = self.lists[0][i]
            self.lists.append(got)
        self.parents = [p for s, n in enumerate(new) for p in (trees[s] if trees and trees[s] is not None else chain(n))]
        self.has_parents = trees is not None
        self.depth, self.sees = [], []
        for f, n in zip(self.first, new):
            depth, sees = [], np.zeros((n, n), bool)
            for i in range(n):
                p = self.parents[f + i]
                depth.append(depth[p] + 1 if p >= 0 else 0)
                if p >= 0:
                    sees[i] = sees[p]
                sees[i, i] = True
            self.depth += depth
            self.sees.append(sees)

    def set(self, hip, batch):
        hip.set_batch(batch, self.context, self.new, [p for l in self.lists for p in l],
                      self.parents if self.has_parents else None)

    def batch(self, hip, cache, heads, spare=0, kernels=0):
        b = hip.alloc_batch(cache, heads, len(self.new) + spare, max(1, self.tokens) + spare, max(1, sum(map(len, self.lists))) + spare)
        take(b, kernels)
        self.set(hip, b)
        return b

    def rows(self, pool, s, kv):
        """Sequence s's keys or values [position][kv_heads][head_dim] of a pool [page][2][row][head][dim]."""
        n = self.context[s] + self.new[s]
        return pool[self.lists[s], kv].reshape(-1, *pool.shape[3:])[:n]

    def place(self, s, position):
        return self.lists[s][position // self.L], position % self.L


def pool_of(r, pages, L, kvh, hd, kv):
    p = r.standard_normal((pages, 2, L, kvh, hd), dtype=np.float32)
    return bf16_to_f32(f32_to_bf16(p)) if kv == TH_KV_BF16 else p


def cache_of(hip, pool, kv):
    c = hip.alloc_paged(pool.shape[0], pool.shape[2], pool.shape[3], pool.shape[4], kv)
    for i, page in enumerate(pool):
        hip.write_paged(c, i, page[0], page[1])
    return c


def read_pool(hip, cache):
    return np.stack([np.stack(hip.read_paged(cache, i)) for i in range(cache.shape[0])])


def buf(hip, a):
    b = hip.alloc(np.asarray(a).size)
    hip.write(b, a)
    return b


def attention64(step, q, pool, heads):
    """Results [token][head][dim], and the bound of each."""
    kvh, hd = pool.shape[3:]
    out, tol = np.empty((step.tokens, heads, hd)), np.empty((step.tokens, heads, hd))
    for s, (c, n, f) in enumerate(zip(step.context, step.new, step.first)):
        if not n:
            continue
        k64, v64 = (step.rows(pool, s, i).astype(np.float64) for i in (0, 1))
        hidden = np.concatenate([np.zeros((n, c), bool), ~step.sees[s]], 1)
        for h in range(heads):
            k, v = k64[:, h * kvh // heads], v64[:, h * kvh // heads]
            x = q[f:f + n, h].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                score = np.where(hidden, -np.inf, x @ k.T / np.sqrt(hd))
                most = np.where(hidden, 0, np.abs(x) @ np.abs(k).T / np.sqrt(hd)).max(1)
            p = np.exp(score - score.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            # What is not seen takes no part, NaN or not.
            seen_v = np.where(hidden.all(0)[:, None], 0, v)
            if np.isnan(seen_v).any() or np.isinf(seen_v).any():
                for i in range(n):
                    out[f + i, h] = p[i][~hidden[i]] @ v[~hidden[i]]
                    tol[f + i, h] = p[i][~hidden[i]] @ np.abs(v[~hidden[i]])
            else:
                out[f:f + n, h], tol[f:f + n, h] = p @ seen_v, p @ np.abs(seen_v)
            d = ((hd + 2) * U + 2.0**-21 + 4 * U) * most
            tol[f:f + n, h] *= 2 * (d + (c + n + 8) * U + 2.0**-21)[:, None]
    return out, tol


def check(got, want, tol, what=""):
    finite = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[~finite & ~np.isnan(want)], want[~finite & ~np.isnan(want)]), what
    off, most = np.abs(got[finite] - want[finite]), tol[finite] + 1e-37
    assert (off <= most).all(), f"{what}: {(off > most).sum()} of {off.size} off, by up to {np.max(off / most)} of the bound"


def run_attention(hip, step, q, pool, heads, kv, kernels=0):
    cache = cache_of(hip, pool, kv)
    batch = step.batch(hip, cache, heads, kernels=kernels)
    bq, out = buf(hip, q), buf(hip, np.full(q.size, 7, np.float32))
    hip.paged_attention(out, bq, cache, batch)
    return hip.read(out).reshape(q.shape)


# (contexts, new tokens): lengths about 16 and 64, sequences without tokens, of one, of many.
LENGTHS = [
    ([0], [1]), ([1], [1]), ([15], [1]), ([16], [1]), ([63], [1]), ([64], [1]), ([65], [1]), ([1000], [1]),
    ([0, 300, 17, 64], [1, 1, 1, 1]), ([5, 40, 7], [0, 1, 0]), ([0], [16]), ([0], [17]), ([30], [5]), ([200, 3], [33, 2]),
    ([0, 120], [150, 70]), ([77, 0, 500], [64, 129, 1]), ([10], [300]),
]
SHAPES = [(16, 8, 128), (32, 8, 128), (4, 2, 128), (8, 1, 128), (3, 3, 64), (16, 1, 64), (6, 2, 128), (10, 2, 256), (4, 4, 256), (7, 1, 128)]


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("lengths", range(len(LENGTHS)))
def test_attention_lengths(hip, lengths, kv, kernels):
    r = np.random.default_rng(lengths)
    heads, kvh, hd = SHAPES[lengths % 3]
    step = Step(r, *LENGTHS[lengths], [16, 32, 64][lengths % 3])
    pool = pool_of(r, step.pages, step.L, kvh, hd, kv)
    q = r.standard_normal((step.tokens, heads, hd), dtype=np.float32)
    check(run_attention(hip, step, q, pool, heads, kv, kernels), *attention64(step, q, pool, heads))


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("page", [16, 256])
@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
def test_attention_shapes(hip, heads, kvh, hd, page, kv, kernels):
    r = np.random.default_rng(heads * 31 + hd + page)
    step = Step(r, [100, 0, 31], [1, 40, 3], page, shared=1)
    pool = pool_of(r, step.pages, page, kvh, hd, kv)
    q = r.standard_normal((step.tokens, heads, hd), dtype=np.float32)
    check(run_attention(hip, step, q, pool, heads, kv, kernels), *attention64(step, q, pool, heads))


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("heads,kvh,hd", [(16, 8, 128), (32, 8, 128), (8, 1, 64), (6, 2, 256)])
@pytest.mark.parametrize("new", [2, 9, 25, 64, 65, 256])
def test_attention_trees(hip, new, heads, kvh, hd, kv, kernels):
    r = np.random.default_rng(new * 7 + heads)
    context, counts = [130, 0, 57], [new, max(1, new // 2), 1]
    trees = [some_tree(r, new, back=new, roots=True), some_tree(r, counts[1]), None]
    step = Step(r, context, counts, 16, trees)
    pool = pool_of(r, step.pages, 16, kvh, hd, kv)
    q = r.standard_normal((step.tokens, heads, hd), dtype=np.float32)
    check(run_attention(hip, step, q, pool, heads, kv, kernels), *attention64(step, q, pool, heads))


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("heads,new", [(16, 5), (32, 30), (32, 90)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38, -1e20])
def test_what_is_not_seen_does_not_count(hip, heads, new, bad, kv, kernels):
    """Rows behind the last position, and drafted tokens of other branches, hold
    NaN, infinities, or numbers beside which the others are nothing."""
    r = np.random.default_rng(new)
    tree = some_tree(r, new)
    step = Step(r, [45, 20], [new, new], 32, [tree, None])
    pool = pool_of(r, step.pages, 32, 8, 128, kv)
    used = np.zeros(pool.shape[:1] + (32,), bool)
    for s in range(2):
        for p in range(step.context[s] + step.new[s]):
            used[step.place(s, p)] = True
    bad = np.float32(bad) if kv == TH_KV_F32 else bf16_to_f32(f32_to_bf16(np.float32([bad])))[0]
    pool.transpose(0, 2, 1, 3, 4)[~used] = bad
    # A tree's token and a chain's: those that do not follow them stay finite.
    for s, i in ((0, new - 2), (1, new - 1)):
        page, row = step.place(s, step.context[s] + i)
        pool[page, :, row, 3] = bad
        pool[page, 1, row, 5, 17] = bad
    q = r.standard_normal((step.tokens, heads, 128), dtype=np.float32)
    want, tol = attention64(step, q, pool, heads)
    group = heads // 8
    touched = np.zeros((step.tokens, heads), bool)
    for s, i in ((0, new - 2), (1, new - 1)):
        touched[step.first[s]:step.first[s] + new, 3 * group:4 * group] |= step.sees[s][:, i:i + 1]
    got = run_attention(hip, step, q, pool, heads, kv, kernels)
    assert np.isfinite(got[~touched][:, :17]).all() and np.isfinite(got[~touched][:, 18:]).all()
    check(got[~touched], want[~touched], tol[~touched])
    # Where a key that is seen has such values, so has the result.
    assert np.isfinite(bad) or not np.isfinite(got[touched]).all(-1).any()


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("new", [1, 20, 70])
@pytest.mark.parametrize("scale", [1e-18, 1e-3, 30.0, 1e15])
def test_attention_of_large_and_small_values(hip, scale, new, kv, kernels):
    """Values and keys far from one: keys times `scale`, queries by its inverse, values by it."""
    r = np.random.default_rng(new)
    step = Step(r, [150], [new], 64)
    pool = pool_of(r, step.pages, 64, 2, 128, TH_KV_F32) * np.float32(scale)
    if kv == TH_KV_BF16:
        pool = bf16_to_f32(f32_to_bf16(pool))
    q = r.standard_normal((step.tokens, 8, 128), dtype=np.float32) / np.float32(scale)
    check(run_attention(hip, step, q, pool, 8, kv, kernels), *attention64(step, q, pool, 8))


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("new", [1, 12, 80])
def test_attention_of_sharp_and_flat_scores(hip, new, kv, kernels):
    """Scores of hundreds (one key has it all) and of zero (an average)."""
    r = np.random.default_rng(new + 5)
    step = Step(r, [333], [new], 16)
    pool = pool_of(r, step.pages, 16, 2, 128, kv)
    q = r.standard_normal((step.tokens, 8, 128), dtype=np.float32)
    q[:, ::2] *= 60
    q[:, 1::4] = 0
    check(run_attention(hip, step, q, pool, 8, kv, kernels), *attention64(step, q, pool, 8))


@gpu
@pytest.mark.parametrize("heads,kvh,context,new,kv", [(16, 8, [33000], [1], TH_KV_F32), (32, 8, [9000], [60], TH_KV_F32),
                                                      (32, 8, [5000, 12, 2100], [7, 1, 300], TH_KV_BF16),
                                                      (8, 8, [20000, 100], [2, 1], TH_KV_BF16), (4, 4, [6000], [256], TH_KV_F32)])
def test_attention_of_long_contexts(hip, heads, kvh, context, new, kv, kernels):
    r = np.random.default_rng(sum(context))
    step = Step(r, context, new, 64, [some_tree(r, n) if n <= 60 else None for n in new])
    pool = pool_of(r, step.pages, 64, kvh, 128, kv)
    q = r.standard_normal((step.tokens, heads, 128), dtype=np.float32)
    check(run_attention(hip, step, q, pool, heads, kv, kernels), *attention64(step, q, pool, heads))


@gpu
def test_attention_past_32_bits(hip):
    """Pages whose offsets pass 2^31 values, and 2^32 bytes."""
    r = np.random.default_rng(1)
    pages, L = 9000, 128
    cache = hip.alloc_paged(pages, L, 8, 128)  # 9.4 GB, 2.4e9 values
    step = Step(r, [300, 40], [3, 70], L, spare=0)
    step.lists = [[8999, 1, 8998], [8500]]
    pool = pool_of(r, 4, L, 8, 128, TH_KV_F32)
    for i, p in enumerate([8999, 1, 8998, 8500]):
        hip.write_paged(cache, p, pool[i, 0], pool[i, 1])
    q = r.standard_normal((73, 16, 128), dtype=np.float32)
    batch = step.batch(hip, cache, 16, kernels=7)
    bq, out = buf(hip, q), hip.alloc(q.size)
    hip.paged_attention(out, bq, cache, batch)
    got = hip.read(out).reshape(q.shape)
    step.lists = [[0, 1, 2], [3]]
    check(got, *attention64(step, q, pool, 16))
    k, v = (r.standard_normal((73, 8, 128), dtype=np.float32) for _ in range(2))
    rope = buf(hip, np.tile(np.float32([1, 0]), 400 * 64))
    hip.paged_append(out, bq, buf(hip, k), buf(hip, v), None, None, rope, cache, batch, EPS)
    assert np.array_equal(hip.read(out).reshape(q.shape), q)
    got_k, got_v = hip.read_paged(cache, 8998)
    assert np.array_equal(got_k[44:47], k[:3]) and np.array_equal(got_v[44:47], v[:3])
    assert np.array_equal(got_k[:44], pool[2, 0, :44]) and np.array_equal(got_k[47:], pool[2, 0, 47:])
    got_k, got_v = hip.read_paged(cache, 8500)
    assert np.array_equal(got_k[40:110], k[3:]) and np.array_equal(got_v[40:110], v[3:])


# ---- append ----

def rope_table(positions, hd, theta=1e6):
    a = np.arange(positions)[:, None] * theta ** (-np.arange(0, hd, 2) / hd)
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def normed_and_rotated64(x, gain, rope, hd):
    x = x.astype(np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(EPS))) * bf16_to_f32(gain).astype(np.float64)
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    c, s = (rope[:, None, :, i].astype(np.float64) for i in (0, 1))
    length = np.abs(a) + np.abs(b)
    return np.concatenate([a * c - b * s, b * c + a * s], -1), np.concatenate([length, length], -1) * (hd + 16) * U


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("heads,kvh,hd,page", [(16, 8, 128, 16), (32, 8, 128, 64), (3, 3, 64, 32), (10, 2, 256, 128), (7, 1, 128, 16)])
@pytest.mark.parametrize("context,new,tree", [([0], [1], False), ([40], [1], False), ([15, 0, 31, 100], [1, 18, 0, 130], False),
                                              ([33, 5], [40, 12], True)])
@pytest.mark.parametrize("norms", ["both", "none", "k"])
def test_append(hip, context, new, tree, heads, kvh, hd, page, norms, kv):
    r = np.random.default_rng(sum(new) + heads)
    step = Step(r, context, new, page, [some_tree(r, n) for n in new] if tree else None)
    pool = pool_of(r, step.pages, page, kvh, hd, kv)
    cache = cache_of(hip, pool, kv)
    batch = step.batch(hip, cache, heads)
    q, k, v = (r.standard_normal((step.tokens, h, hd), dtype=np.float32) * np.float32(3) for h in (heads, kvh, kvh))
    gq, gk = (f32_to_bf16(1 + 0.3 * r.standard_normal(hd).astype(np.float32)) for _ in range(2))
    gq, gk = (gq if norms == "both" else None), (gk if norms != "none" else None)
    up = lambda g: None if g is None else hip.upload(Tensor((hd,), g))  # noqa: E731
    rope = rope_table(max(c + n for c, n in zip(context, new)), hd)
    bq, bk, bv, out = buf(hip, q), buf(hip, k), buf(hip, v), hip.alloc(q.size)
    wq, wk, table = up(gq), up(gk), buf(hip, rope)
    hip.paged_append(out, bq, bk, bv, wq, wk, table, cache, batch, EPS)
    position = np.repeat(context, new) + step.depth
    want, tol = normed_and_rotated64(q, gq, rope[position], hd)
    check(hip.read(out).reshape(q.shape), want, tol)
    assert np.array_equal(hip.read(bq), q.reshape(-1)) and np.array_equal(hip.read(bk), k.reshape(-1))
    want, tol = normed_and_rotated64(k, gk, rope[position], hd)
    got = read_pool(hip, cache)
    left = np.ones((step.pages, page), bool)
    for s in range(len(new)):
        for i in range(new[s]):
            t, at = step.first[s] + i, step.place(s, context[s] + i)
            left[at] = False
            more = 2.0**-8 * np.abs(want[t]) * (1 + 2.0**-8) if kv == TH_KV_BF16 else 0
            check(got[at[0], 0, at[1]], want[t], tol[t] * 1.01 + more)
            assert np.array_equal(got[at[0], 1, at[1]], bf16_to_f32(f32_to_bf16(v[t])) if kv == TH_KV_BF16 else v[t])
    assert np.array_equal(got.transpose(0, 2, 1, 3, 4)[left], pool.transpose(0, 2, 1, 3, 4)[left])
    # In place.
    hip.paged_append(bq, bq, bk, bv, wq, wk, table, cache, batch, EPS)
    assert np.array_equal(hip.read(bq), hip.read(out))


@gpu
def test_append_matches_the_device_calls(hip):
    """A chain alone: q/k rmsnorm, rope and copy, then attention, of the trait's
    calls over contiguous caches (n products more or less in the sums: 1e-6)."""
    r = np.random.default_rng(3)
    heads, kvh, hd, n, ctx = 16, 8, 128, 21, 50
    step = Step(r, [ctx], [n], 16)
    pool = pool_of(r, step.pages, 16, kvh, hd, TH_KV_F32)
    cache = cache_of(hip, pool, TH_KV_F32)
    batch = step.batch(hip, cache, heads)
    q, k, v = (r.standard_normal((n, h, hd), dtype=np.float32) for h in (heads, kvh, kvh))
    gain = hip.upload(Tensor((hd,), f32_to_bf16(1 + 0.1 * r.standard_normal(hd).astype(np.float32))))
    rope = buf(hip, rope_table(ctx + n, hd))
    out, res = hip.alloc(q.size), hip.alloc(q.size)
    hip.paged_append(out, buf(hip, q), buf(hip, k), buf(hip, v), gain, gain, rope, cache, batch, EPS)
    hip.paged_attention(res, out, cache, batch)
    tq, tk, tv = buf(hip, q), buf(hip, k), buf(hip, v)
    for x, h in ((tq, heads), (tk, kvh)):
        hip.rmsnorm(x, gain, EPS)
        hip.rope(x, rope, ctx, h, hd)
    caches = []
    for i, x in ((0, tk), (1, tv)):
        b = hip.alloc((ctx + n) * kvh * hd)
        old = np.zeros((ctx + n, kvh, hd), np.float32)
        old[:ctx] = step.rows(pool, 0, i)[:ctx]
        hip.write(b, old)
        hip.copy(b, ctx * kvh * hd, x, 0, n * kvh * hd)
        caches.append(b)
    other = hip.alloc(q.size)
    hip.attention(other, tq, *caches, ctx, heads, hd, kvh)
    a, b = hip.read(out), hip.read(tq)
    assert np.max(np.abs(a - b)) <= 1e-6 * np.max(np.abs(b))
    a, b = hip.read(res), hip.read(other)
    # th_attention's own terms are of 16 bits.
    assert np.linalg.norm(a - b) <= 2e-5 * np.linalg.norm(b)


# ---- verification and moved rows ----

def accept_of(step, logits, tokens):
    picks, n_kept, kept = logits.argmax(1), [], np.full(step.tokens, -1)
    for f, n in zip(step.first, step.new):
        path = [0] if n else []
        while path:
            at = [i for i in range(1, n) if step.parents[f + i] == path[-1] and tokens[f + i] == picks[f + path[-1]]]
            if not at:
                break
            path.append(at[0])
        n_kept.append(len(path))
        kept[f:f + len(path)] = path
    return picks, np.array(n_kept), kept


@gpu
@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 1000, 1001, 4096, 4099, 8193, 40001, 151936])
@pytest.mark.parametrize("new", [[1], [5, 0, 9], [30, 17, 1, 64]])
def test_accept(hip, new, vocab):
    r = np.random.default_rng(vocab + sum(new))
    step = Step(r, [10] * len(new), new, 16, [some_tree(r, n, back=3, roots=True) for n in new])
    cache = hip.alloc_paged(step.pages, 16, 1, 64)
    batch = step.batch(hip, cache, 1)
    logits = r.standard_normal((step.tokens, vocab), dtype=np.float32)
    logits[0, vocab // 2:] = logits[0].max()  # a tie: the lowest index
    picks = logits.argmax(1)
    tokens = r.integers(0, vocab, step.tokens)
    for s, f in enumerate(step.first):
        for i in range(1, new[s]):
            if step.parents[f + i] >= 0 and r.random() < 0.8:
                tokens[f + i] = picks[f + step.parents[f + i]]
    for got, want in zip(hip.accept(batch, buf(hip, logits), tokens), accept_of(step, logits, tokens)):
        assert np.array_equal(got, want)


@gpu
def test_accept_orders_as_argmax(hip):
    r = np.random.default_rng(2)
    rows = r.standard_normal((6, 5000)).astype(np.float32)
    rows[0, 77] = np.nan
    rows[1, 4999] = np.inf
    rows[2] = -np.inf
    rows[3] = -0.0
    rows[3, 100] = 0.0
    rows[4] = -np.nan
    step = Step(r, [0], [6], 16)
    batch = step.batch(hip, hip.alloc_paged(step.pages, 16, 1, 64), 1)
    picks, _, _ = hip.accept(batch, buf(hip, rows), np.zeros(6, np.uint32))
    assert list(picks) == [hip.argmax(buf(hip, x)) for x in rows]


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("layers,kvh,hd,page,context,new", [
    (1, 8, 128, 16, [0], [1]), (3, 8, 128, 16, [9, 0, 30], [24, 16, 40]), (70, 1, 64, 32, [5], [20]),
    (2, 2, 64, 16, list(range(70)), [8] * 70), (2, 3, 256, 64, [11, 3], [256, 200])])
def test_keep(hip, layers, kvh, hd, page, context, new, kv):
    r = np.random.default_rng(layers + sum(new))
    step = Step(r, context, new, page)
    pools = [pool_of(r, step.pages, page, kvh, hd, kv) for _ in range(layers)]
    caches = [cache_of(hip, p, kv) for p in pools]
    batch = step.batch(hip, caches[0], kvh)
    kept, counts = np.full(step.tokens, -1, np.int32), []
    for s, (f, n) in enumerate(zip(step.first, new)):
        # All, none, every other one, or any.
        some = [np.arange(n), np.arange(0), np.arange(1, n, 2), np.sort(r.permutation(n)[:r.integers(0, n + 1)])][(s + 3) % 4 if n < 200 else 2]
        kept[f:f + len(some)] = some
        counts.append(len(some))
    want = [p.copy() for p in pools]
    for s, (f, c) in enumerate(zip(step.first, context)):
        for before, after in zip(pools, want):
            for j in range(counts[s]):
                (p0, r0), (p1, r1) = step.place(s, c + kept[f + j]), step.place(s, c + j)
                after[p1, :, r1] = before[p0, :, r0]
    hip.paged_keep(caches, batch, counts, kept)
    for c, w in zip(caches, want):
        assert np.array_equal(read_pool(hip, c), w)


# ---- graphs ----

@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("at", [([100, 7], [60, 13]), ([2] * 73, [1] * 73)])
def test_captured_calls_take_any_step(hip, at, kv, kernels):
    """One graph of an append and an attention, captured with two trees or with
    73 single tokens, over steps of other lengths, pages and trees, with the same
    calls run eagerly between the replays."""
    r = np.random.default_rng(8)
    heads, kvh, hd, page = 16, 8, 128, 16
    lens = [at, ([3, 900], [1, 2]), ([500], [70]), ([0, 0, 0], [20, 1, 1]), ([64], [1]), ([], []), ([1200, 40], [5, 66])]
    steps = [Step(r, c, n, page, [some_tree(r, x) for x in n] if i % 2 == 0 else None, spare=0) for i, (c, n) in enumerate(lens)]
    most, tokens = max(s.pages for s in steps), 73
    pool = pool_of(r, most, page, kvh, hd, kv)
    cache = cache_of(hip, pool, kv)
    batch = hip.alloc_batch(cache, heads, 73, tokens + 1, most)
    take(batch, kernels)
    q, k, v = (r.standard_normal((tokens, h, hd), dtype=np.float32) for h in (heads, kvh, kvh))
    bq, bk, bv = buf(hip, q), buf(hip, k), buf(hip, v)
    gain = hip.upload(Tensor((hd,), f32_to_bf16(1 + 0.1 * r.standard_normal(hd).astype(np.float32))))
    rope = buf(hip, rope_table(1500, hd))
    turned, out = hip.alloc(q.size), hip.alloc(q.size)
    steps[0].set(hip, batch)
    calls = lambda o, t, x, y, z: (hip.paged_append(t, x, y, z, gain, gain, rope, cache, batch, EPS), hip.paged_attention(o, t, cache, batch))  # noqa: E731
    hip.graph_begin()
    calls(out, turned, bq, bk, bv)
    graph = hip.graph_end()
    for again in range(3):
        for i, step in enumerate(steps):
            step.set(hip, batch)
            hip.write(out, np.full(q.size, 5, np.float32))
            graph.launch()
            got = hip.read(out).reshape(q.shape)
            assert (got[step.tokens:] == 5).all(), "rows behind the last token"
            now = [buf(hip, x[:step.tokens]) for x in (q, q, q, k, v)]
            calls(*now)
            eager = hip.read(now[0]).reshape(-1, heads, hd)
            assert np.array_equal(got[:step.tokens], eager), (again, i)
            if again == 0:
                pool = read_pool(hip, cache)
                check(got[:step.tokens], *attention64(step, hip.read(now[1]).reshape(-1, heads, hd), pool, heads))
    with pytest.raises(InvalidArgument, match="captured"):
        hip.set_batch(batch, [0], [tokens + 1], list(range(-(-(tokens + 1) // page))))
    graph.free()


@gpu
def test_two_captured_batches_of_calls(hip, kernels):
    """A graph captured with a long and a short sequence and one with 21 single
    tokens, over one batch and tables of 100 and 102 positions: both take any
    step that is set later, in turn and with eager calls between, and none is
    set whose replay would read past a table or have more tokens."""
    r = np.random.default_rng(18)
    heads, kvh, hd, page, tokens = 16, 8, 128, 16, 30
    steps = [Step(r, c, n, page, None, spare=0) for c, n in [([20, 3], [25, 5]), ([99], [1]), ([0, 70], [3, 18]), ([4] * 21, [1] * 21)]]
    most = max(s.pages for s in steps)
    pool = pool_of(r, most, page, kvh, hd, TH_KV_F32)
    cache = cache_of(hip, pool, TH_KV_F32)
    batch = hip.alloc_batch(cache, heads, 21, tokens, most)
    take(batch, kernels)
    q, k, v = (r.standard_normal((tokens, h, hd), dtype=np.float32) for h in (heads, kvh, kvh))
    rope, long_rope = buf(hip, rope_table(100, hd)), buf(hip, rope_table(102, hd))
    graphs = []
    for step, table in [(steps[0], rope), (steps[3], long_rope)]:
        step.set(hip, batch)
        x = [buf(hip, a[:step.tokens]) for a in (q, k, v)]
        out = hip.alloc(len(x[0]))
        hip.graph_begin()
        hip.paged_append(x[0], x[0], x[1], x[2], None, None, table, cache, batch, EPS)
        hip.paged_attention(out, x[0], cache, batch)
        graphs.append((hip.graph_end(), x, out))
    for again in range(2):
        for step in steps[:0:-1] if again else steps[1:]:
            step.set(hip, batch)
            now = [buf(hip, a[:step.tokens]) for a in (q, k, v)]
            eager = hip.alloc(len(now[0]))
            hip.paged_append(now[0], now[0], now[1], now[2], None, None, rope, cache, batch, EPS)
            hip.paged_attention(eager, now[0], cache, batch)
            want = hip.read(eager)
            for graph, x, out in graphs:
                hip.write(x[0], q.ravel()[:len(x[0])])
                graph.launch()
                assert np.array_equal(hip.read(out)[:want.size], want)
    for context, new, what in [([100], [1], "position 100"), ([98, 99], [1, 2], "position 100"), ([0], [22], "captured with this batch at 21")]:
        with pytest.raises(InvalidArgument, match=what):
            hip.set_batch(batch, context, new, range(sum(-(-(c + n) // page) for c, n in zip(context, new))))
    for graph, *_ in graphs:
        graph.free()


# ---- refusals ----

@gpu
def test_refusals(hip):
    bad = pytest.raises(InvalidArgument)
    for args in [(0, 16, 1, 128, 0), (4, 8, 1, 128, 0), (4, 48, 1, 128, 0), (4, 512, 1, 128, 0), (4, 16, 0, 128, 0), (4, 16, 1025, 128, 0),
                 (4, 16, 1, 96, 0), (4, 16, 1, 128, 2), (1 << 27, 16, 1, 128, 0)]:
        with pytest.raises(InvalidArgument):
            hip.alloc_paged(*args)
    cache, other = hip.alloc_paged(4, 16, 2, 128), hip.alloc_paged(5, 16, 2, 128)
    assert cache.shape == (4, 16, 2, 128, TH_KV_F32)
    for args in [(3, 1, 1, 1), (0, 1, 1, 1), (34, 1, 1, 1), (4, 0, 1, 1), (4, 1, 0, 1), (4, 1, 1, 0), (4, 65537, 1, 1), (4, 1, 1 << 23, 1)]:
        with pytest.raises(InvalidArgument):
            hip.alloc_batch(cache, *args)
    for f in (lambda: hip.read_paged(cache, 4), lambda: hip.write_paged(cache, 4, np.zeros(16 * 256), np.zeros(16 * 256))):
        with pytest.raises(InvalidArgument):
            f()
    with pytest.raises(ValueError):
        hip.write_paged(cache, 0, np.zeros(3), np.zeros(3))
    batch = hip.alloc_batch(cache, 4, 3, 40, 4)
    hip.set_batch(batch, [3], [2], [1])
    buffers = {n: hip.alloc(n) for n in (2 * 512, 2 * 256, 3 * 512, 512)}
    q, kv, rope = buffers[1024], buffers[512], hip.alloc(5 * 128)
    out = hip.alloc(1024)
    hip.paged_append(out, q, kv, kv, None, None, rope, cache, batch, EPS)
    gains = hip.upload(Tensor((64,), np.zeros(64)))
    for f in [lambda: hip.paged_append(out, buffers[1536], kv, kv, None, None, rope, cache, batch, EPS),
              lambda: hip.paged_append(buffers[1536], q, kv, kv, None, None, rope, cache, batch, EPS),
              lambda: hip.paged_append(out, q, q, kv, None, None, rope, cache, batch, EPS),
              lambda: hip.paged_append(out, q, kv, q, None, None, rope, cache, batch, EPS),
              lambda: hip.paged_append(out, q, kv, kv, gains, None, rope, cache, batch, EPS),
              lambda: hip.paged_append(out, q, kv, kv, None, gains, rope, cache, batch, EPS),
              lambda: hip.paged_append(out, q, kv, kv, None, None, hip.alloc(4 * 128), cache, batch, EPS),
              lambda: hip.paged_append(out, q, kv, kv, None, None, rope, other, batch, EPS),
              lambda: hip.paged_attention(q, q, cache, batch), lambda: hip.paged_attention(kv, q, cache, batch),
              lambda: hip.paged_attention(out, q, other, batch),
              lambda: hip.accept(batch, hip.alloc(7), [0, 0]), lambda: hip.accept(batch, hip.alloc(0), [0, 0]),
              lambda: hip.paged_keep([cache, cache], batch, [1], [1, -1]), lambda: hip.paged_keep([cache, other], batch, [1], [1, -1]),
              lambda: hip.paged_keep([cache, hip.alloc_paged(4, 16, 2, 128, TH_KV_BF16)], batch, [1], [1, -1]),
              lambda: hip.paged_keep([cache], batch, [3], [0, 1]), lambda: hip.paged_keep([cache], batch, [2], [1, 0]),
              lambda: hip.paged_keep([cache], batch, [2], [0, 0]), lambda: hip.paged_keep([cache], batch, [1], [2, -1]),
              lambda: hip.paged_keep([cache], batch, [1], [-1, -1])]:
        with pytest.raises(InvalidArgument):
            f()
    with pytest.raises(ValueError):
        hip.accept(batch, hip.alloc(8), [0])
    with pytest.raises(ValueError):
        hip.set_batch(batch, [-1], [2], [1])
    with pytest.raises(TypeError):
        hip.set_batch(batch, [0.5], [2], [1])
    # Another device's stream would not wait for the batch.
    second = Hip(0)
    with pytest.raises(InvalidArgument, match="belongs"):
        second.paged_attention(out, q, cache, batch)
    with pytest.raises(InvalidArgument, match="belongs"):
        second.set_batch(batch, [3], [2], [1])
    second.close()
    hip.graph_begin()
    try:
        for f in (lambda: hip.alloc_paged(4, 16, 2, 128), lambda: hip.alloc_batch(cache, 4, 1, 1, 1), lambda: hip.read_paged(cache, 0),
                  lambda: hip.write_paged(cache, 0, np.zeros(16 * 256), np.zeros(16 * 256)), lambda: hip.set_batch(batch, [3], [2], [1]),
                  lambda: hip.accept(batch, kv, [0, 0]), lambda: hip.paged_keep([cache], batch, [1], [1, -1])):
            with pytest.raises(InvalidArgument):
                f()
        with pytest.raises(RuntimeError):
            cache.free()
        hip.paged_attention(out, q, cache, batch)
    finally:
        hip.graph_end().free()


@gpu
def test_batches_of_nothing(hip):
    cache = hip.alloc_paged(2, 16, 2, 128)
    batch = hip.alloc_batch(cache, 4, 2, 4, 2)
    none, rope = hip.alloc(0), hip.alloc(128)
    for set_it in (lambda: None, lambda: hip.set_batch(batch, [], [], []), lambda: hip.set_batch(batch, [20, 0], [0, 0], [1, 0])):
        set_it()
        hip.paged_append(none, none, none, none, None, None, rope, cache, batch, EPS)
        hip.paged_attention(none, none, cache, batch)
        picks, n_kept, kept = hip.accept(batch, none, [])
        assert not picks.size and not kept.size and not n_kept.any()
        hip.paged_keep([cache], batch, n_kept, kept)
    hip.synchronize()

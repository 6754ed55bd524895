"""What th_batch_set refuses, lays out and plans (include/titania_hip_test_paged.h),
without a GPU: bad pages and counts, tokens' places and what a tree's see, and
the attention's items, which cover every row and position once and stay within
the room that launches and partial results have."""

from __future__ import annotations

import ctypes as C
import math
import random

import numpy as np
import pytest

from titania_amd import InvalidArgument
from titania_amd._lib import LIB_PATH, check

ROWS = [16, 128, 256]  # of a tile, by class
ALL = 7
SLAB_FLOATS = 1024 * 128 * (128 + 2)  # of partial results
SPLIT_BLOCKS = 2048  # the most of a class's blocks where it is split


def batch_set(context, new, pages, parents=None, cache=(64, 16, 2, 128), bf16=False, heads=4, room=(8, 400, 64), classes=ALL,
              captured=1 << 62, table=1 << 62):
    f = C.CDLL(str(LIB_PATH)).th_test_batch_set
    f.argtypes = [C.c_void_p, C.c_uint, C.c_size_t, C.c_size_t, C.c_size_t, C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p,
                  C.c_void_p, C.c_void_p, C.c_void_p, C.POINTER(C.c_size_t), C.c_void_p, C.POINTER(C.c_size_t), C.c_void_p]
    shape = (C.c_size_t * 9)(*cache, int(bf16), heads, *room)
    c, n, p = (np.array(x, np.uint32) for x in (context, new, pages))
    t = None if parents is None else np.array(parents, np.int32)
    total = int(n.sum(dtype=np.int64)) if n.sum(dtype=np.int64) < 1 << 20 else 0
    tokens, tree = np.zeros((total, 4), np.uint32), np.zeros((total, 4), np.uint64)
    most = total * 16 + 4 * len(new) + 4 * SPLIT_BLOCKS
    items, joins, first = np.zeros((most, 9), np.uint32), np.zeros((most, 6), np.uint32), np.zeros(4, np.uint32)
    n_items, n_joins = C.c_size_t(most), C.c_size_t(most)
    check(f(shape, classes, captured, table, len(c), c.ctypes.data, n.ctypes.data, p.ctypes.data, len(p),
            None if t is None else t.ctypes.data, tokens.ctypes.data, tree.ctypes.data, items.ctypes.data, C.byref(n_items), joins.ctypes.data, C.byref(n_joins),
            first.ctypes.data))
    return tokens, tree, items[:n_items.value], joins[:n_joins.value], first


@pytest.mark.parametrize("what,args", [
    ("past the end of 2 pages", dict(context=[32], new=[1], pages=[0, 1])),
    ("3 pages for sequences of 2", dict(context=[31], new=[1], pages=[0, 1, 2])),
    ("page 64 at index 1", dict(context=[31], new=[1], pages=[0, 64])),
    ("page 4294967295", dict(context=[31], new=[1], pages=[0, 0xffffffff])),
    ("9 sequences", dict(context=[0] * 9, new=[1] * 9, pages=range(9))),
    ("401 tokens", dict(context=[0], new=[401], pages=range(26))),
    ("65 pages", dict(context=[0] * 5, new=[1] * 5, pages=[0] * 65)),
    ("past the end", dict(context=[0xffffffff], new=[1], pages=range(64))),
    ("past the end", dict(context=[0xffffffff], new=[0xffffffff], pages=range(64))),
    ("new rows in two places", dict(context=[5, 7], new=[1, 1], pages=[3, 3])),
    ("new rows in two places", dict(context=[5], new=[30], pages=[3, 4, 3])),
    ("in the context of sequence 1", dict(context=[5, 17], new=[1, 1], pages=[3, 3, 4])),
    ("in the context of sequence 0", dict(context=[17], new=[1], pages=[3, 3])),
    ("parent -2 of token 0", dict(context=[0], new=[2], pages=[0], parents=[-2, 0])),
    ("parent 1 of token 1", dict(context=[0], new=[2], pages=[0], parents=[-1, 1])),
    ("parent 0 of token 0 of sequence 1", dict(context=[0, 0], new=[2, 1], pages=[0, 1], parents=[-1, 0, 0])),
    ("a tree of 257 tokens", dict(context=[0], new=[257], pages=range(17), parents=[-1] * 257)),
    ("captured with this batch at 9", dict(context=[0], new=[10], pages=[0], captured=9)),
    ("position 40: a graph", dict(context=[3, 40, 0], new=[1, 1, 2], pages=[0, 1, 2, 3, 4], table=40)),
    ("position 12: a graph", dict(context=[10], new=[4], pages=[0], parents=[-1, 0, 1, 0], table=12)),
    ("position 13: a graph", dict(context=[10], new=[4], pages=[0], parents=[-1, 0, 1, 2], table=13)),
    ("1073741825 positions of sequence 1", dict(context=[0, 1 << 30], new=[1, 1], pages=[1] + [0] * ((1 << 22) + 1),
                                                cache=(64, 256, 2, 128), room=(8, 400, 1 << 23))),
])
def test_refused(what, args):
    with pytest.raises(InvalidArgument, match=what):
        batch_set(**args)


def test_allowed():
    batch_set([], [], [])
    batch_set([40, 0], [0, 0], [1, 1, 1])  # sequences without tokens read and write nothing
    batch_set([32, 35, 32], [1, 0, 2], [7, 8, 1, 7, 8, 1, 7, 8, 2])  # shared contexts
    batch_set([0], [400], range(25), parents=[i - 1 for i in range(400)])  # a chain, however long
    batch_set([0], [256], range(16), parents=[-1] * 256)
    batch_set([0], [9], [0], captured=9)
    batch_set([3, 39, 60], [1, 1, 0], range(8), captured=2, table=40)  # what has no tokens is not rotated
    batch_set([10], [4], [0], parents=[-1, 0, 1, 0], table=13)
    batch_set([(1 << 30) - 1], [1], [0] * ((1 << 22) - 1) + [1], cache=(64, 256, 2, 128), room=(8, 400, 1 << 23))


def test_tokens_and_trees():
    r = random.Random(1)
    for _ in range(60):
        seqs = r.randint(1, 5)
        context, new = [r.choice([0, 15, 16, r.randint(0, 100)]) for _ in range(seqs)], [r.choice([0, 1, r.randint(1, 70)]) for _ in range(seqs)]
        counts = [-(-(c + n) // 16) for c, n in zip(context, new)]
        order = r.sample(range(64), sum(counts)) if sum(counts) <= 64 else None
        if order is None:
            continue
        parents = [r.randint(-1, i - 1) if r.random() < 0.5 else i - 1 for n in new for i in range(n)]
        tokens, tree, *_ = batch_set(context, new, order, parents)
        t = at = 0
        for s in range(seqs):
            mine, depth, sees = order[at:at + counts[s]], [], []
            chain = all(p == i - 1 for i, p in enumerate(parents[t:t + new[s]]))
            for i in range(new[s]):
                p, place = parents[t + i], context[s] + i
                depth.append(depth[p] + 1 if p >= 0 else 0)
                sees.append((sees[p] if p >= 0 else 0) | 1 << i)
                assert list(tokens[t + i]) == [mine[place // 16] * 16 + place % 16, context[s] + depth[i], s, i]
                if not chain:
                    assert sum(int(w) << 64 * k for k, w in enumerate(tree[t + i])) == sees[i]
            t, at = t + new[s], at + counts[s]


def log_int(r, low, high):
    return min(high, int(math.exp(r.uniform(math.log(low), math.log(high + 1)))))


@pytest.mark.parametrize("seed", range(40))
def test_plans(seed):
    r = random.Random(seed)
    heads, kvh = r.choice([(16, 8), (32, 8), (8, 1), (16, 1), (3, 3), (64, 64), (1024, 1024), (7, 1), (6, 2)])
    hd, group = r.choice([64, 128, 128, 256]), heads // kvh
    seqs, page = log_int(r, 1, 200), 256
    context = [log_int(r, 1, r.choice([50, 5000, 300000])) - 1 for _ in range(seqs)]
    new = [r.choice([0, 1, 1, log_int(r, 1, r.choice([4, 60, 3000]))]) for _ in range(seqs)]
    while sum(new) * heads > 1 << 21:
        new = [n // 2 for n in new]
    counts = [-(-(c + n) // page) for c, n in zip(context, new)]
    classes = r.choice([ALL, ALL, 1, 3, 5])
    tokens, _, items, joins, first = batch_set(
        context, new, np.arange(sum(counts)), cache=(sum(counts) + 1, page, kvh, hd), bf16=r.random() < 0.5, heads=heads,
        room=(seqs, max(1, sum(new)), max(1, sum(counts))), classes=classes)
    token0 = {sum(new[:s]): s for s in range(seqs) if new[s]}
    covered, slabs = {}, np.zeros(SLAB_FLOATS // (16 * (hd + 2)) + 1, int)
    parts = {}
    assert first[0] == 0 and first[-1] == len(items) and all(np.diff(first.astype(int)) >= 0)
    for c in range(3):
        assert first[c] == first[c + 1] or (classes >> c & 1 and (hd < 256 or c == 0))
        mine = items[first[c]:first[c + 1]].astype(int)
        lengths = mine[:, 7] - mine[:, 6]
        assert (np.diff(lengths) <= 0).all()  # the longest first
        if c:
            rows = sum(new) * group
            assert len(mine) * kvh <= (rows // 17 + rows // 128 + 2) * kvh + SPLIT_BLOCKS
        for t0, n, ctx, page0, is_tree, row0, k0, k1, part in mine:
            s = token0[t0]
            assert (n, ctx, page0, is_tree) == (new[s], context[s], sum(counts[:s]), 0) and row0 % ROWS[c] == 0
            rows = min(ROWS[c], n * group - row0)
            last = ctx + (row0 + rows - 1) // group + 1
            assert rows > 0 and 0 <= k0 < k1 <= last and k0 % 64 == 0 and (k1 % 64 == 0 or k1 == last)
            covered.setdefault((s, row0, rows, last), []).append((k0, k1))
            if part == 0xffffffff:
                assert (k0, k1) == (0, last)
            else:
                each = ROWS[c] // 16 * kvh
                slabs[part:part + each] += 1
                parts.setdefault((t0, row0), []).append((part, each, ROWS[c] // 16, rows))
    assert slabs.max() <= 1 and slabs[-1] == 0
    done = {s: 0 for s in token0.values()}
    for (s, row0, rows, last), ranges in covered.items():
        ranges.sort()
        assert ranges[0][0] == 0 and ranges[-1][1] == last and all(a[1] == b[0] for a, b in zip(ranges, ranges[1:]))
        done[s] += rows
    assert done == {s: new[s] * group for s in token0.values()}
    assert len(joins) == len(parts)
    for t0, rows, row0, part, n_parts, each_head in joins.astype(int):
        mine = sorted(parts.pop((t0, row0)))
        assert len(mine) == n_parts > 1 and [p for p, *_ in mine] == [part + i * mine[0][1] for i in range(n_parts)]
        assert all(m[2] == each_head and m[3] == rows for m in mine)

"""Paged caches where a step's calls meet others: steps set without waiting for
the ones before, two device handles at once, as many heads as a batch takes, and
Python's checks of what it passes on."""

from __future__ import annotations

import numpy as np
import pytest

from test_paged import EPS, Step, attention64, buf, cache_of, check, pool_of, rope_table, some_tree, take
from titania_amd import TH_KV_BF16, TH_KV_F32, Hip

gpu = pytest.mark.gpu


@gpu
def test_steps_that_nothing_waits_for(hip):
    """Steps of other lengths, set and enqueued one after another on one batch,
    give what each gives alone: a set waits until the one before is copied."""
    r = np.random.default_rng(21)
    heads, kvh, hd, page = 16, 8, 128, 16
    lens = [([900, 3], [40, 1]), ([4000], [1]), ([0, 70, 5], [3, 18, 1]), ([2500], [60]), ([], []), ([1], [1])] * 4
    steps = [Step(r, c, n, page, [some_tree(r, x) for x in n], spare=0) for c, n in lens]
    most = max(s.pages for s in steps)
    pool = pool_of(r, most, page, kvh, hd, TH_KV_F32)
    cache = cache_of(hip, pool, TH_KV_F32)
    batch = hip.alloc_batch(cache, heads, 4, 100, most)
    queries = [buf(hip, r.standard_normal((s.tokens, heads, hd), dtype=np.float32)) for s in steps]
    outs = [hip.alloc(len(q)) for q in queries]
    hip.synchronize()
    for step, q, out in zip(steps, queries, outs):
        step.set(hip, batch)
        hip.paged_attention(out, q, cache, batch)
    got = [hip.read(out) for out in outs]
    for step, q, out, x in zip(steps, queries, outs, got):
        step.set(hip, batch)
        hip.paged_attention(out, q, cache, batch)
        assert np.array_equal(hip.read(out), x)
    check(got[0].reshape(-1, heads, hd), *attention64(steps[0], hip.read(queries[0]).reshape(-1, heads, hd), pool, heads))


@gpu
def test_two_handles_at_once(hip):
    """Batches of two device handles of one GPU over one cache: their streams run
    side by side, each with partial results of its own."""
    r = np.random.default_rng(22)
    heads, kvh, hd, page = 16, 8, 128, 32
    other = Hip(0)
    step = Step(r, [6000, 50], [30, 1], page, None, spare=0)
    pool = pool_of(r, step.pages, page, kvh, hd, TH_KV_BF16)
    cache = cache_of(hip, pool, TH_KV_BF16)
    qs = [r.standard_normal((step.tokens, heads, hd), dtype=np.float32) for _ in range(2)]
    devices = [hip, other]
    batches = [step.batch(d, cache, heads) for d in devices]
    bufs = [buf(d, q) for d, q in zip(devices, qs)]
    outs = [[d.alloc(q.size) for _ in range(8)] for d, q in zip(devices, qs)]
    hip.synchronize()
    other.synchronize()
    for i in range(8):
        for d in (0, 1):
            devices[d].paged_attention(outs[d][i], bufs[d], cache, batches[d])
    for d in (0, 1):
        first = devices[d].read(outs[d][0])
        check(first.reshape(qs[d].shape), *attention64(step, qs[d], pool, heads))
        assert all(np.array_equal(devices[d].read(o), first) for o in outs[d][1:])
    batches[1].free()
    for b in [bufs[1]] + outs[1]:
        b.free()
    other.close()


@gpu
@pytest.mark.parametrize("seqs,new", [(65536, 16), (1 << 10, 1 << 10)])
def test_as_many_heads_as_a_batch_takes(hip, seqs, new):
    """2^24 heads, in 65536 sequences of 16 tokens and in 1024 of 1024: 64
    sequences again and again, whose results are the first ones' bits."""
    r = np.random.default_rng(23)
    heads, kvh, hd, page, same = 16, 8, 64, 16, 64
    per = -(-new // page)
    cache = hip.alloc_paged(seqs * per, page, kvh, hd, TH_KV_BF16)
    batch = hip.alloc_batch(cache, heads, seqs, seqs * new, seqs * per)
    take(batch, 7)
    pages = np.arange(seqs * per, dtype=np.uint32)[::-1]
    hip.set_batch(batch, np.zeros(seqs, np.uint32), np.full(seqs, new, np.uint32), pages)
    q, k, v = (r.standard_normal((same, new, h, hd), dtype=np.float32) for h in (heads, kvh, kvh))

    def again(a):
        b = hip.alloc(seqs // same * a.size)
        hip.write(b, np.tile(a.ravel(), seqs // same))
        return b

    bq, bk, bv = again(q), again(k), again(v)
    rope = buf(hip, rope_table(new, hd))
    hip.paged_append(bq, bq, bk, bv, None, None, rope, cache, batch, EPS)
    for b in (bk, bv):
        b.free()
    out = hip.alloc(len(bq))
    hip.paged_attention(out, bq, cache, batch)
    got = hip.read(out).reshape(seqs // same, -1)
    assert (got == got[0]).all()
    turned = hip.read(bq).reshape(seqs // same, -1)
    assert (turned == turned[0]).all()
    for b in (bq, out):
        b.free()
    # One sequence of them in 64 bits, from the cache's rows.
    step = Step(r, [0], [new], page, None, spare=0)
    step.lists = [list(range(per))]
    at = int(r.integers(same))
    pool = np.stack([np.stack(hip.read_paged(cache, int(p))) for p in pages[at * per:(at + 1) * per]])
    check(got[0].reshape(same, new, heads, hd)[at], *attention64(step, turned[0].reshape(same, new, heads, hd)[at], pool, heads))
    batch.free()
    cache.free()


@pytest.mark.parametrize("values,error", [([0.5], TypeError), ([-1], ValueError), ([1 << 32], ValueError), ([float("nan")], TypeError)])
def test_whole_numbers(values, error):
    from titania_amd.device import _ints

    with pytest.raises(error):
        _ints(values, np.uint32)

"""What captured calls ask of later steps of their batch, and for how long."""

from __future__ import annotations

import numpy as np
import pytest

from test_paged import EPS, Step, buf, cache_of, pool_of, rope_table
from titania_amd import TH_KV_BF16, TH_KV_F32, Hip, InvalidArgument
from titania_amd._lib import check, lib

gpu = pytest.mark.gpu
HEADS, KVH, HD, PAGE = 32, 8, 128, 16


class Batch:
    """A batch over pages in order, and the calls that a graph of it holds."""

    def __init__(self, hip, r, tokens=200, kv=TH_KV_F32):
        self.hip, self.r = hip, r
        step = Step(r, [0], [600], PAGE, spare=0)
        self.pool = pool_of(r, step.pages, PAGE, KVH, HD, kv)
        self.cache = cache_of(hip, self.pool, kv)
        self.batch = hip.alloc_batch(self.cache, HEADS, 4, tokens, step.pages)
        self.tokens = tokens
        self.q, self.k = (r.standard_normal((tokens, h, HD), dtype=np.float32) for h in (HEADS, KVH))

    def set(self, context, new):
        self.hip.set_batch(self.batch, [context], [new], range(-(-(context + new) // PAGE)))

    def refuses(self, what, context, new):
        with pytest.raises(InvalidArgument, match=what):
            self.set(context, new)

    def capture(self, context, new, positions, end=True):
        """A graph of an append over a table of `positions` and an attention, and its buffers."""
        self.set(context, new)
        x = [buf(self.hip, a[:new]) for a in (self.q, self.k, self.k)] + [buf(self.hip, rope_table(positions, HD)), self.hip.alloc(new * HEADS * HD)]
        self.hip.graph_begin()
        self.hip.paged_append(x[0], x[0], x[1], x[2], None, None, x[3], self.cache, self.batch, EPS)
        self.hip.paged_attention(x[4], x[0], self.cache, self.batch)
        return (self.hip.graph_end() if end else None), x

    def attention(self, context, new):
        self.set(context, new)
        q, out = buf(self.hip, self.q[:new]), self.hip.alloc(new * HEADS * HD)
        self.hip.paged_attention(out, q, self.cache, self.batch)
        return self.hip.read(out)


@gpu
@pytest.mark.parametrize("order", [(0, 1, 2), (2, 1, 0), (1, 2, 0)])
def test_a_graph_asks_as_long_as_it_is_there(hip, order):
    """Three graphs of one batch, freed in any order: what is refused are the
    steps that one of those left cannot take."""
    b = Batch(hip, np.random.default_rng(1))
    limits = [(50, 400), (20, 300), (30, 200)]  # tokens, positions
    graphs = [None] * 3
    for i in (0, 2, 1):  # (each with no more tokens than those before it)
        graphs[i] = b.capture(100, *limits[i])
    for gone in range(4):
        left = [limits[i] for i in order[gone:]]
        most, end = (min(x) for x in zip(*left)) if left else (b.tokens, 600)
        b.set(0, most)
        b.set(end - 1, 1)
        if left:
            b.refuses(f"captured with this batch at {most}", 0, most + 1)
            b.refuses(f"position {end}", end, 1)
        for i in order[gone:]:
            b.set(40, 2)
            graphs[i][0].launch()
        hip.synchronize()
        if left:
            graphs[order[gone]][0].free()


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
def test_the_plan_is_its_own_again(hip, kv):
    """Kernels that a graph does not hold are planned for once it is freed: the
    bits of 150 tokens are those of a batch that no graph was captured with."""
    other, few = (Batch(hip, np.random.default_rng(2), kv=kv) for _ in range(2))
    hip.set_batch(few.batch, [3] * 4, [1] * 4, range(4))
    q, out = buf(hip, few.q[:4]), hip.alloc(4 * HEADS * HD)
    hip.graph_begin()
    hip.paged_attention(out, q, few.cache, few.batch)
    graph = hip.graph_end()
    few.refuses("captured", 0, 5)
    assert np.array_equal(few.attention(300, 4), other.attention(300, 4))
    graph.free()
    assert np.array_equal(few.attention(300, 150), other.attention(300, 150))


@gpu
def test_batches_outlive_graphs_and_devices():
    """A capture that ends with its device asks nothing of anybody, and batches
    may be freed in any order."""
    dev = Hip(0)
    r = np.random.default_rng(3)
    batches = [Batch(dev, r) for _ in range(3)]
    graph, x = batches[0].capture(0, 3, 100)
    batches[1].batch.free()
    batches[0].refuses("captured", 0, 4)
    graph.free()
    batches[0].set(0, 4)
    batches[2].set(0, 4)
    batches[2].capture(0, 3, 100, end=False)
    dev.close()
    for b in (batches[2], batches[0]):
        lib().th_batch_free(None, b.batch.handle)
        b.batch.handle = None


@gpu
def test_a_batch_is_replayed_on_its_own_stream(hip):
    """Another device's stream would not wait for a set: a graph with a batch's
    calls is refused there, one of other calls is not."""
    b = Batch(hip, np.random.default_rng(4))
    other = Hip(0)
    graph, x = b.capture(0, 3, 100)
    hip.graph_begin()
    hip.add(x[1], x[2])
    plain = hip.graph_end()
    hip.write(x[1], np.zeros(len(x[1])))
    with pytest.raises(InvalidArgument, match="captured with"):
        check(lib().th_graph_launch(other.handle, graph.handle))
    check(lib().th_graph_launch(other.handle, plain.handle))
    other.synchronize()
    assert np.array_equal(hip.read(x[1]), b.k[:3].ravel())
    graph.launch()
    hip.synchronize()
    for g in (graph, plain):
        g.free()
    other.close()


@gpu
def test_one_graph_of_two_batches(hip):
    """What a graph asks of two batches ends for both; for one that is freed
    before it there is nothing left to end."""
    r = np.random.default_rng(5)
    for gone in (None, 0, 1):
        batches = [Batch(hip, r) for _ in range(2)]
        x = [[buf(hip, a[:n]) for a in (b.q, b.k, b.k)] for b, n in zip(batches, (4, 9))]
        rope = buf(hip, rope_table(50, HD))
        for b, n in zip(batches, (4, 9)):
            b.set(10, n)
        hip.graph_begin()
        for b, (q, k, v) in zip(batches, x):
            hip.paged_append(q, q, k, v, None, None, rope, b.cache, b.batch, EPS)
        graph = hip.graph_end()
        for b, n in zip(batches, (4, 9)):
            b.refuses(f"captured with this batch at {n}", 0, n + 1)
            b.refuses("position 50", 50, 1)
            b.set(49, 1)
        graph.launch()
        hip.synchronize()
        if gone is not None:
            batches[gone].batch.free()
        graph.free()
        for i, b in enumerate(batches):
            if i != gone:
                b.set(0, 100)
                b.set(300, 1)

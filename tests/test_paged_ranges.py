"""Attention over paged caches whose values differ widely in size from place to
place: what a token does not see, and how a plan cuts the positions, changes no
result. Compared with float64 under test_paged's bounds."""

from __future__ import annotations

import numpy as np
import pytest

from test_paged import Step, attention64, check, kernels, pool_of, run_attention  # noqa: F401 (a fixture)
from titania_amd import TH_KV_BF16, TH_KV_F32
from titania_amd.synth import bf16_to_f32, f32_to_bf16

gpu = pytest.mark.gpu


def branches(*lengths):
    """A tree of branches that all follow the context: each a chain."""
    return [-1 if i == 0 else sum(lengths[:b]) + i - 1 for b, n in enumerate(lengths) for i in range(n)]


def scaled(step, pool, kv, factors):
    """The pool with the values of sequence 0's drafted token i times factors[i]."""
    for i, f in enumerate(factors):
        page, row = step.place(0, step.context[0] + i)
        pool[page, 1, row] *= np.float32(f)
    return bf16_to_f32(f32_to_bf16(pool)) if kv == TH_KV_BF16 else pool


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("context", [0, 64, 128, 6400])
@pytest.mark.parametrize("lengths,factors", [
    ((64, 30), (2.0**20, 1)), ((64, 30), (2.0**40, 1)), ((64, 30), (1e20, 1)), ((64, 30), (1, 1e20)), ((64, 30), (2.0**-20, 1)),
    ((64, 64, 64, 20), (2.0**30, 2.0**20, 2.0**10, 1)), ((64, 64, 128), (1, 1e20, 1)), ((30, 100), (1e20, 1)),
], ids=str)
@pytest.mark.parametrize("hd", [64, 128])
def test_branches_of_other_sizes(hip, hd, lengths, factors, context, kv, kernels):  # noqa: F811
    """Branches of a tree, of which the first fills whole 64 positions, whose
    values are larger or smaller than other branches' by so much that together
    they have no scale: each branch's results are its own."""
    r = np.random.default_rng(sum(lengths) + context)
    step = Step(r, [context], [sum(lengths)], 32, [branches(*lengths)])
    pool = scaled(step, pool_of(r, step.pages, 32, 2, hd, TH_KV_F32), kv, np.repeat(factors, lengths))
    q = r.standard_normal((step.tokens, 8, hd), dtype=np.float32)
    check(run_attention(hip, step, q, pool, 8, kv, kernels), *attention64(step, q, pool, 8))


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("context", [0, 64])
@pytest.mark.parametrize("large", [2.0**40, 1e20])
def test_one_large_value_among_zeros(hip, large, context, kv, kernels):  # noqa: F811
    """A branch of zeros and one large value, then an ordinary one."""
    r = np.random.default_rng(context)
    step = Step(r, [context], [90], 32, [branches(64, 26)])
    factors = np.ones(90)
    factors[:64] = 0
    factors[63] = large
    pool = scaled(step, pool_of(r, step.pages, 32, 2, 128, TH_KV_F32), kv, factors)
    q = r.standard_normal((step.tokens, 8, 128), dtype=np.float32)
    check(run_attention(hip, step, q, pool, 8, kv, kernels), *attention64(step, q, pool, 8))


def flat_scores(hip, size, signs, new, context, kv, kernels):
    """Averages of thousands of values whose sums f32 does not hold, of one sign
    or both, where a plan splits the positions."""
    r = np.random.default_rng(new + context)
    step = Step(r, [context], [new], 64)
    pool = pool_of(r, step.pages, 64, 2, 128, TH_KV_F32)
    pool[:, 1] = r.uniform(0.1, 1, pool[:, 1].shape) * size
    if signs:
        pool[:, 1] *= r.choice([-1, 1], pool[:, 1].shape)
    pool = bf16_to_f32(f32_to_bf16(pool)) if kv == TH_KV_BF16 else pool
    q = np.float32(0.01) * r.standard_normal((step.tokens, 8, 128), dtype=np.float32)
    check(run_attention(hip, step, q, pool, 8, kv, kernels), *attention64(step, q, pool, 8))


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("context", [2000, 6400])
@pytest.mark.parametrize("new", [1, 20, 70])
@pytest.mark.parametrize("size,signs", [(1e33, True), (1e34, False), (1e35, True)])
def test_flat_scores_over_large_values(hip, size, signs, new, context, kv, kernels):  # noqa: F811
    """(Sums with weights of at most one are in range: the kernel for few rows has those.)"""
    flat_scores(hip, size, signs, new, context, kv, kernels)


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("context", [2000, 6400])
@pytest.mark.parametrize("new", [20, 70])
@pytest.mark.parametrize("large_tiles", [7, 5])
def test_flat_scores_over_values_near_the_largest(hip, large_tiles, new, context, kv):
    """The kernels for many rows, where sums are past f32's range and averages are not."""
    flat_scores(hip, 3e38, False, new, context, kv, large_tiles)


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("context,new", [([20000], [1]), ([40000] + [400] * 9, [16] * 10)])
def test_joins_of_more_parts_than_lanes(hip, context, new, kv, kernels):  # noqa: F811
    """One KV head, so that the chip is filled by one long sequence's parts:
    hundreds of a few rows, and of many beside others of two."""
    r = np.random.default_rng(len(context))
    step = Step(r, context, new, 256)
    pool = pool_of(r, step.pages, 256, 1, 128, kv)
    q = r.standard_normal((step.tokens, 16, 128), dtype=np.float32)
    check(run_attention(hip, step, q, pool, 16, kv, kernels), *attention64(step, q, pool, 16))


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("what", [0, 1])
@pytest.mark.parametrize("heads,kvh,first,new", [(32, 8, 64, 128), (512, 256, 128, 256)])
def test_what_all_rows_see_is_not_taken_one_by_one(hip, what, heads, kvh, first, new, kv):
    """A prompt with a position whose key, or values, are 2^-14 of its
    neighbours': the tokens of later tiles, all of which see it, get the bits that
    they get when the positions before them are their context. (Tiles of 256 rows
    of so few positions, or so many heads, that no plan splits either.)"""
    r = np.random.default_rng(first + what)
    step = Step(r, [0], [new], 32, spare=0)
    after = Step(r, [first], [new - first], 32, spare=0)
    after.lists = step.lists
    pool = pool_of(r, step.pages, 32, kvh, 128, TH_KV_F32)
    page, row = step.place(0, 20)
    pool[page, what, row] *= np.float32(2.0**-14)
    pool = bf16_to_f32(f32_to_bf16(pool)) if kv == TH_KV_BF16 else pool
    q = r.standard_normal((new, heads, 128), dtype=np.float32)
    got = run_attention(hip, step, q, pool, heads, kv, 7)
    check(got, *attention64(step, q, pool, heads))
    same = got[first:] == run_attention(hip, after, q[first:], pool, heads, kv, 7)
    assert same.all(), f"{(~same).sum()} of {same.size} differ"


@gpu
@pytest.mark.parametrize("kv", [TH_KV_F32, TH_KV_BF16])
@pytest.mark.parametrize("what", [0, 1])
@pytest.mark.parametrize("factor", [2.0**8, 2.0**11, 2.0**-11])
@pytest.mark.parametrize("context", [0, 50])
def test_branches_of_sizes_that_have_a_scale(hip, context, factor, what, kv, kernels):  # noqa: F811
    """Keys or values of another branch up to 2^13 times a token's own take as
    many of the bits of 2^-38 that its terms leave out: 2^-25 of the largest
    that it sees, for each value as it is, for each key times the query's."""
    r = np.random.default_rng(int(abs(np.log2(factor))) + context)
    step = Step(r, [context], [100], 32, [branches(64, 36)])
    pool = pool_of(r, step.pages, 32, 2, 128, TH_KV_F32)
    for i in range(64):
        page, row = step.place(0, context + i)
        pool[page, what, row] *= np.float32(factor)
    pool = bf16_to_f32(f32_to_bf16(pool)) if kv == TH_KV_BF16 else pool
    q = r.standard_normal((100, 8, 128), dtype=np.float32)
    want, tol = attention64(step, q, pool, 8)
    sees = np.concatenate([np.ones((100, context), bool), step.sees[0]], 1)
    largest = np.array([np.abs(step.rows(pool, 0, what)[s]).max((0, 2)) for s in sees])  # [token][KV head]
    largest = np.repeat(largest, 4, 1).astype(np.float64)
    if what:
        tol += 2.0**-25 * largest[:, :, None]
    else:
        value = np.array([np.abs(step.rows(pool, 0, 1)[s]).max((0, 2)) for s in sees])
        d = 2.0**-25 * largest * np.abs(q).sum(-1) / np.sqrt(128)
        tol += 2 * (d * np.repeat(value, 4, 1))[:, :, None]
    check(run_attention(hip, step, q, pool, 8, kv, kernels), want, tol)

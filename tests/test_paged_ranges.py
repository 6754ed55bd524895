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
def test_branches_of_other_sizes(hip, lengths, factors, context, kv, kernels):  # noqa: F811
    """Branches of a tree, of which the first fills whole 64 positions, whose
    values are larger or smaller than other branches' by so much that together
    they have no scale: each branch's results are its own."""
    r = np.random.default_rng(sum(lengths) + context)
    step = Step(r, [context], [sum(lengths)], 32, [branches(*lengths)])
    pool = scaled(step, pool_of(r, step.pages, 32, 2, 128, TH_KV_F32), kv, np.repeat(factors, lengths))
    q = r.standard_normal((step.tokens, 8, 128), dtype=np.float32)
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

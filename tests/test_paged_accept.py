"""The verification of drafted tokens at its largest: rows whose parts are as many
as a launch takes, and more rows than one launch's results have room for."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from test_paged import Step, accept_of, buf
from titania_amd._lib import LIB_PATH
from titania_amd._lib import check as ok

gpu = pytest.mark.gpu
MOST_PICKS = 1 << 17  # that a launch leaves in pinned memory


def parts_of(rows, cols):
    f = C.CDLL(str(LIB_PATH)).th_test_accept_parts
    f.argtypes = [C.c_size_t, C.c_size_t, *[C.POINTER(C.c_size_t)] * 3]
    out = [C.c_size_t() for _ in range(3)]
    ok(f(rows, cols, *map(C.byref, out)))
    return [x.value for x in out]


@pytest.mark.parametrize("rows", [1, 2, 3, 24, 462, 2047, 2048, 2049, 65535, MOST_PICKS - 1, MOST_PICKS, MOST_PICKS + 1, 1 << 24])
def test_no_part_is_empty(rows):
    """A part without values leaves nothing, and would be waited for as if it were late."""
    for cols in [1, 3, 4, 5, 4095, 4096, 4097, 151936, 1 << 20, (1 << 22) + 1, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, (1 << 23) + 4097,
                 (1 << 24) + 5, (1 << 32) - 2]:
        at_once, splits, part = parts_of(rows, cols)
        assert 0 < at_once <= rows and at_once * splits <= MOST_PICKS
        assert part % 4 == 0 and (splits - 1) * part < cols <= splits * part


@gpu
@pytest.mark.parametrize("cols", [(1 << 22) + 1, (1 << 23) + 1, (1 << 23) + 4097])
@pytest.mark.parametrize("at", [0, 1 << 21, -1])
def test_one_row_of_many_parts(hip, cols, at):
    logits = np.random.default_rng(cols).standard_normal((1, cols), dtype=np.float32)
    logits[0, at] = 20
    step = Step(np.random.default_rng(1), [0], [1], 16)
    batch = step.batch(hip, hip.alloc_paged(step.pages, 16, 1, 64), 1)
    picks, n_kept, kept = hip.accept(batch, buf(hip, logits), [7])
    assert list(picks) == [at % cols] and list(n_kept) == [1] and list(kept) == [0]


@gpu
def test_more_rows_than_a_launch_takes(hip):
    """140000 drafted tokens over a vocabulary of five, in two launches."""
    r = np.random.default_rng(3)
    new = [20000] * 7
    step = Step.__new__(Step)  # (what each token sees is not needed here, and would be 400 MB a sequence)
    step.new, step.first, step.tokens = new, [sum(new[:s]) for s in range(7)], sum(new)
    step.parents = [i - 1 for n in new for i in range(n)]
    per = -(-20000 // 256)
    cache = hip.alloc_paged(7 * per, 256, 1, 64)
    batch = hip.alloc_batch(cache, 1, 7, step.tokens, 7 * per)
    hip.set_batch(batch, [0] * 7, new, range(7 * per))
    assert step.tokens > MOST_PICKS
    logits = r.standard_normal((step.tokens, 5), dtype=np.float32)
    tokens = r.integers(0, 5, step.tokens)
    picks = logits.argmax(1)
    for s in (0, 6):  # the first and the last accept most of what follows
        f = step.first[s]
        tokens[f + 1:f + 200] = picks[f:f + 199]
    for got, want in zip(hip.accept(batch, buf(hip, logits), tokens), accept_of(step, logits, tokens)):
        assert np.array_equal(got, want)

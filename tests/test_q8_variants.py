"""Which kernels the tested products of 8-bit rows take: every one that a call
can reach, each tile whole and with K split where the estimate splits it."""

from __future__ import annotations

import ctypes as C
import math
import random

import pytest

import test_q8
from titania_amd import InvalidArgument
from titania_amd._lib import LIB_PATH, check

# Tall tiles with K split, which test_q8's products leave out.
TALL_SPLIT = [(386, 3373, 21902), (387, 6776, 14237), (305, 8112, 15815), (524, 5421, 22361)]

FEW, TILES = range(7), range(7, 18)
TWO_A_CU = 9  # the tile whose ring is short, for many tiles; a split has few
REACHED = {(v, False) for v in [*FEW, *TILES]} | {(v, True) for v in TILES if v != TWO_A_CU}


def variant(n, rows, cols):
    """(variant, whether K is split) of th_matmul_q8."""
    which, ksplit = C.c_int(), C.c_int()
    f = C.CDLL(str(LIB_PATH)).th_test_matmul_q8_variant
    f.argtypes = [C.c_size_t] * 3 + [C.POINTER(C.c_int)] * 2
    check(f(n, rows, cols, C.byref(which), C.byref(ksplit)))
    return which.value, ksplit.value > 1


def test_products_take_every_variant():
    assert {variant(*p) for p in test_q8.PRODUCTS + TALL_SPLIT} == REACHED


def test_no_product_takes_another():
    r = random.Random(2)
    for most in ((20000, 200000, 131071), (1 << 25, 1 << 25, 131071)):
        for _ in range(15000):
            shape = [max(1, int(math.exp(r.uniform(0, math.log(m))))) for m in most]
            assert variant(*shape) in REACHED, shape


@pytest.mark.parametrize("n,rows,cols", [(0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 131072), ((1 << 25) + 1, 1, 1)])
def test_no_size_has_no_variant(n, rows, cols):
    with pytest.raises(InvalidArgument):
        variant(n, rows, cols)


@pytest.mark.gpu
@pytest.mark.parametrize("n,rows,cols", TALL_SPLIT)
def test_matmul_of_tall_split_tiles(hip, n, rows, cols):
    test_q8.test_matmul(hip, n, rows, cols)

"""8-bit rows at their largest: as many as a handle takes."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from test_q8 import buf, repeated, rows64
from titania_amd._lib import LIB_PATH, check

MOST_ROWS = 1 << 25


def dequantize_threads(rows, cols):
    threads = C.c_size_t()
    f = C.CDLL(str(LIB_PATH)).th_test_dequantize_q8_threads
    f.argtypes = [C.c_size_t, C.c_size_t, C.POINTER(C.c_size_t)]
    check(f(rows, cols, C.byref(threads)))
    return threads.value


@pytest.mark.parametrize("rows,cols", [(1, 1), (17, 300), (8192, 2560), (MOST_ROWS, 1), (MOST_ROWS, 513), (MOST_ROWS, 1793),
                                       (MOST_ROWS - 16, 1800), (1 << 21, 24000), (440000, 131071), (MOST_ROWS, 131071)])
def test_launches_stay_below_2_to_32_threads(rows, cols):
    """A launch of more is refused by the runtime. (1793 columns of all rows
    are 305 GB with their f32 values: the smallest that was past it.)"""
    threads = dequantize_threads(rows, cols)
    assert 0 < threads < 1 << 32
    # One launch as long as it can be one: 256 threads for every 16 rows x 256 columns.
    whole = (rows + 15) // 16 * ((cols + 255) // 256) * 256
    assert threads == whole or threads > 1 << 29


@pytest.mark.gpu
def test_dequantize_in_several_launches(hip):
    rows, cols = MOST_ROWS, 513
    first = (1 << 22) // 3 * 16  # rows of the first launch
    assert dequantize_threads(rows, cols) == first // 16 * 3 * 256
    x = np.random.default_rng(17).standard_normal((19, cols)).astype(np.float32)
    q, out, one = hip.alloc_q8(rows, cols), hip.alloc(rows * cols), hip.alloc(40 * cols)
    hip.quantize_q8(q, repeated(hip, x, rows))
    hip.dequantize_q8(out, q)
    want_q, want_s = rows64(x)
    want = want_q.astype(np.float32) * want_s[:, None]
    for at in (0, first - 20, rows - 40):
        hip.copy(one, 0, out, at * cols, 40 * cols)
        assert np.array_equal(hip.read(one).reshape(40, cols), want[np.arange(at, at + 40) % 19]), at

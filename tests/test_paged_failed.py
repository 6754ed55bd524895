"""What a batch holds after a set that was refused or that the GPU failed, without
a GPU (include/titania_hip_test_paged.h)."""

from __future__ import annotations

import ctypes as C
import types

import numpy as np
import pytest

from titania_amd import HipError, InvalidArgument, device
from titania_amd._lib import LIB_PATH, TH_ERR_HIP, TH_ERR_INVALID, check


def test_nothing_is_set_after_a_set_that_failed():
    f = C.CDLL(str(LIB_PATH)).th_test_batch_set_failed
    f.argtypes = [C.c_void_p, C.c_size_t, C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]
    context, new = np.array([4000, 3], np.uint32), np.array([1, 40], np.uint32)
    pages = np.arange(251 + 3, dtype=np.uint32)
    shape = (C.c_size_t * 9)(300, 16, 8, 128, 0, 32, 2, 41, 300)
    left = np.full(9, 77, np.uintp)
    with pytest.raises(HipError, match="setting a batch failed") as e:
        check(f(shape, 2, context.ctypes.data, new.ctypes.data, pages.ctypes.data, len(pages), left.ctypes.data))
    assert e.value.code == TH_ERR_HIP and not left.any()


@pytest.mark.parametrize("code,left", [(TH_ERR_INVALID, (1, 2)), (TH_ERR_HIP, (0, 0))])
def test_python_knows_what_is_set(monkeypatch, code, left):
    """The arrays that accept() hands over are of these sizes."""
    results = [0, code]
    monkeypatch.setattr(device, "lib", lambda: types.SimpleNamespace(th_batch_set=lambda *_: results.pop(0)))
    hip = object.__new__(device.Hip)
    hip.handle = None
    batch = device.Batch(hip, None)
    hip.set_batch(batch, [3], [2], [0])
    assert (batch.n_seqs, batch.n_tokens) == (1, 2)
    with pytest.raises(InvalidArgument if code == TH_ERR_INVALID else HipError):
        hip.set_batch(batch, [3, 4], [2, 5], [0, 1])
    assert (batch.n_seqs, batch.n_tokens) == left

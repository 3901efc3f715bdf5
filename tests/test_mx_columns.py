"""The columns that the groups of the few-rows product take, on the host: the function that the
kernel calls (csrc/mx_columns.hpp), for every group of a launch.  None of this reaches a GPU."""
import ctypes as C
import os

import numpy as np
import pytest

LIB = os.path.join(os.path.dirname(os.path.abspath(__file__)), "c", "libmx_columns.so")


@pytest.mark.parametrize("nt", [1, 2])
def test_every_column_is_one_groups(nt):
    """Rows of w inside it; each column stored once, from its own row; the workspace's vectors of four at
    multiples of 16 bytes, inside their row."""
    assert os.path.exists(LIB), "build tests/c first (__graft_entry__.build())"
    host = C.CDLL(LIB)
    for N in [*range(1, 200), 255, 256, 265, 1030, 4099, 5000, 50257]:
        stored, off = np.zeros(N + 64, np.int32), C.c_int()
        outside = host.mx_columns(N, nt, C.c_void_p(stored.ctypes.data), C.byref(off))
        assert outside == 0 and off.value == 0, (N, outside, off.value)
        assert (stored[:N] == 1).all() and not stored[N:].any(), N

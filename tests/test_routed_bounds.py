"""What the routed 8-bit operators' C entries refuse by size, shown without a GPU: the host's checks need a handle to read, not a
device, so a block of zeros stands for one (device 0).  An entry that lets such a call pass goes on to the device and fails otherwise."""
import ctypes

import pytest

from stlq_b200 import operators

torch = pytest.importorskip("torch")

I, L, V = ctypes.c_int, ctypes.c_int64, ctypes.c_void_p
EINVAL = 1
MOST = 2**31 - 4096  # columns of a row


@pytest.fixture
def lib():
    lib = operators._ready()[0]
    lib.stlq_b200_quantize_rows.argtypes = [V, V, I, L, L, I, V, L, V, V]
    lib.stlq_b200_dispatch.argtypes = [V, V, I, L, L, I, I, V, V, I, V, L, V]
    lib.stlq_b200_dispatch_i8.argtypes = [V, V, I, L, L, I, I, V, V, I, V, L, V, V]
    lib.stlq_b200_combine.argtypes = [V, V, I, L, L, I, I, V, I, V, V, I, V, L, V]
    lib.stlq_b200_combine_backward.argtypes = [V, V, I, L, V, L, L, I, I, V, I, V, V, I, V, L, V, V]
    return lib


@pytest.mark.parametrize("cols", [MOST + 1, 2**31 - 256, 2**31 - 1])
def test_rows_whose_column_counters_would_overflow(lib, cols):
    """A thread counts a block's worth past a row's end; from 2^31 - 4095 columns on that may leave 32 bits and come back negative."""
    handle = ctypes.create_string_buffer(4096)
    h, p, ld = ctypes.addressof(handle), 4096, 2**31
    calls = [
        lambda: lib.stlq_b200_quantize_rows(h, p, 0, ld, 1, cols, p, ld, p, None),
        lambda: lib.stlq_b200_dispatch(h, p, 1, ld, 1, cols, 1, p, p, 1, p, ld, None),
        lambda: lib.stlq_b200_dispatch_i8(h, p, 2, ld, 1, cols, 1, p, p, 1, p, ld, p, None),
        lambda: lib.stlq_b200_combine(h, p, 2, ld, 1, cols, 1, None, 0, p, p, 1, p, ld, None),
        lambda: lib.stlq_b200_combine_backward(h, p, 2, ld, p, ld, 1, cols, 1, p, 0, p, p, 1, p, ld, p, None),
    ]
    for call in calls:
        assert call() == EINVAL
        assert b"2^31 - 4096" in lib.stlq_b200_last_error()

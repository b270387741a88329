"""The attribute network on the host, where its parts meet: what is passed on and what is refused, without a GPU."""
import ctypes as C
import os

import pytest

from tinygs_amd import _lib


def test_only_muon_takes_copies():
    from tinygs_amd.optim import create_optimizer
    with pytest.raises(RuntimeError, match="writes no copies"):
        create_optimizer("simple_adam", None, None, copies=[])


@pytest.mark.parametrize("size", [2, 4])
def test_loads_of_row_blocks_end_with_the_matrix(size):
    """The many-row linear kernel reads blocks of 64 rows in pieces of 16 bytes: none passes the matrix's last element,
    however few elements a row has and rows follow the block, and all elements of the block are reached."""
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    f = _lib.load()._ZN3tgs17linear_rows_reachEllll
    f.argtypes, f.restype = [C.c_int64] * 4, C.c_int64
    for cols in list(range(1, 34)) + [127, 128]:
        for stride in {cols, cols + 1, cols + 3, cols + 8}:
            for left in list(range(1, 150)) + [64 * 1000, 64 * 1000 + 1]:
                reach = f(left, cols, stride, size)
                held = min(left, 64)
                assert ((held - 1) * stride + cols) * size <= reach <= ((left - 1) * stride + cols) * size

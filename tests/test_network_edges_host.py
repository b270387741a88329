"""The attribute network on the host, where its parts meet: what is passed on and what is refused, without a GPU."""
import ctypes as C
import glob
import os
import re

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


def test_asm_puts_m0_back():
    """m0 is reserved: the compiler takes no clobber of it, and keeps what it holds there over asm. A statement that
    writes it saves it first and restores it last."""
    found = 0
    for path in sorted(glob.glob(os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc", "*.h*"))):
        for text in re.findall(r"\basm\b[^;]*?\((.*?)\);", open(path).read(), re.S):
            steps = "".join(re.findall(r'"((?:[^"\\]|\\.)*)"', text)).replace("\\n", "\n").replace("\\t", "").split("\n")
            if any(re.match(r"s_mov_b32 m0\b", s) for s in steps):
                found += 1
                assert steps[0] == "s_mov_b32 %0, m0" and re.match(r"s_mov_b32 m0, %0", steps[-1]), (path, steps)
    assert found >= 1


# threads that a launch holds; with more, what is above is lost without an error
LAUNCH = 1 << 32


def test_wide_layer_norm_launches_hold_their_threads():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    f = _lib.load()._ZN3tgs22layer_norm_wide_blocksEl
    f.argtypes, f.restype = [C.c_int64], C.c_int64
    for rows in (1, 65535, 65537, 1 << 22, (1 << 31) - 1):
        assert 1 <= f(rows) <= rows and f(rows) * 1024 < LAUNCH


@pytest.mark.parametrize("count,fits", [(511, True), (512, False)])
def test_muon_refuses_more_than_a_launch_holds(count, fits):
    """Matrices of one row and 2^21 - 1 columns are 2^15 patches of 256 threads each. Their addresses are never read."""
    lib, n = _lib.load(), (1 << 21) - 1

    def array(slot):
        return (_lib.tgs_matrix * count)(*[_lib.tgs_matrix((1 << 40) * (slot + 1) + (1 << 23) * k, 1, n, n,
                                                           _lib.TGS_DTYPE_FLOAT32) for k in range(count)])
    h = C.c_void_p()
    rc = lib.tgs_muon_create(array(0), array(1), array(2), None, count, C.byref(h))
    if fits:
        assert rc == 0 and lib.tgs_muon_destroy(h) == 0
    else:
        assert rc == _lib.TGS_ERR_INVALID and "too large for one step" in lib.tgs_last_error().decode()


BASE = 1 << 20   # addresses that nothing reads: every call below is refused


def refusal(x, w, y, residual=None):
    """What a linear forward is refused for whose preact is y's own matrix: that, where nothing before it is."""
    lib, h = _lib.load(), C.c_void_p()
    assert lib.tgs_network_create(C.byref(h)) == 0
    try:
        assert lib.tgs_linear_forward(h, x, w, None, 0, residual, y, y, None) == _lib.TGS_ERR_INVALID
        return lib.tgs_last_error().decode()
    finally:
        lib.tgs_network_destroy(h)


def test_a_single_row_between_anothers_columns():
    """One row of a buffer's column range beside the rows of another range of it (16 floats a row): a single row's own
    stride says nothing, as callers that hold one row pass its length."""
    def mat(row, col, rows, cols, stride=16):
        return _lib.tgs_matrix(BASE + 4 * (16 * row + col), rows, cols, stride, _lib.TGS_DTYPE_FLOAT32)
    x = _lib.tgs_matrix(BASE * 4, 1, 8, 8, _lib.TGS_DTYPE_FLOAT32)
    for stride in (6, 7, 16):
        for row in (0, 3, 5):
            w = mat(0, 0, 6, 8)
            assert refusal(x, w, mat(row, 8, 1, 6, stride)) == "preact overlaps y"
            assert refusal(x, w, mat(row, 10, 1, 6, stride)) == "preact overlaps y"
            assert refusal(x, w, mat(row, 7, 1, 6, stride)) == "y overlaps w"
            assert refusal(x, mat(0, 8, 6, 8), mat(row, 2, 1, 6, stride)) == "preact overlaps y"
            assert refusal(x, mat(0, 8, 6, 8), mat(row, 3, 1, 6, stride)) == ("y overlaps w" if row < 6 else "preact overlaps y")
    # past the last row, and a row longer than the distance between rows
    assert refusal(x, mat(0, 0, 6, 8), mat(6, 0, 1, 6, 6)) == "preact overlaps y"
    long = _lib.tgs_matrix(BASE + 4 * 8, 1, 20, 20, _lib.TGS_DTYPE_FLOAT32)
    wide = _lib.tgs_matrix(BASE, 20, 8, 16, _lib.TGS_DTYPE_FLOAT32)
    assert refusal(x, wide, long) == "y overlaps w"
    # over the residual: its own matrix, whatever the two strides of the single row say
    apart = _lib.tgs_matrix(BASE * 8, 6, 8, 8, _lib.TGS_DTYPE_FLOAT32)
    y = mat(3, 8, 1, 6, 6)
    assert refusal(x, apart, y, mat(3, 8, 1, 6, 16)) == "preact overlaps residual"
    assert refusal(x, apart, y, mat(3, 9, 1, 6, 16)) == "y overlaps residual"

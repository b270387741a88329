"""What the gradients' clipping takes from the host: the time to bind many matrices, overlaps among them, and numbers that
are not Python's own."""
import ctypes as C
import time

import numpy as np
import pytest
import torch

from tinygs_amd import _lib

F32, F16 = _lib.TGS_DTYPE_FLOAT32, _lib.TGS_DTYPE_FLOAT16


def create(grads, clipped=None):
    """Addresses that nothing reads: nothing is launched."""
    h = C.c_void_p()
    n = len(grads)
    rc = _lib.load().tgs_gradient_clip_create((_lib.tgs_matrix * n)(*grads),
                                              None if clipped is None else (_lib.tgs_matrix * n)(*clipped), n, C.byref(h))
    return rc, h


def words():
    return _lib.load().tgs_last_error().decode()


def test_many_matrices():
    """4096 matrices and as many outputs, in any order: bound in milliseconds, not by holding each against all."""
    n = 4096
    order = np.random.default_rng(1).permutation(2 * n)
    mats = [_lib.tgs_matrix((1 << 20) + int(k) * 4096, 4, 256, 256, F32) for k in order]
    start = time.perf_counter()
    rc, h = create(mats[:n], mats[n:])
    assert rc == 0
    assert time.perf_counter() - start < 1.0
    assert _lib.load().tgs_gradient_clip_destroy(h) == 0


@pytest.mark.parametrize("at, of", [(0, 1), (17, 4000), (4095, 0), (2048, 2047)])
@pytest.mark.parametrize("sets", ["gg", "gc", "cc"])
def test_one_overlap_among_many(at, of, sets):
    n = 4096
    grads = [_lib.tgs_matrix((1 << 20) + k * 4096, 4, 256, 256, F32) for k in range(n)]
    clipped = [_lib.tgs_matrix((1 << 30) + k * 4096, 4, 256, 256, F32) for k in range(n)]
    one, two = (grads if sets[0] == "g" else clipped), (grads if sets[1] == "g" else clipped)
    one[at].data = two[of].data + 4092   # its last element
    rc, _ = create(grads, clipped)
    assert rc == _lib.TGS_ERR_INVALID
    names = {"g": "grads", "c": "clipped"}
    if sets == "gc":
        assert words().endswith(f"clipped[{of}] overlaps grads[{at}]")
    else:
        assert words().endswith(f"{names[sets[0]]}[{max(at, of)}] overlaps {names[sets[0]]}[{min(at, of)}]")


def test_interleaved_columns():
    """Column ranges of one buffer share no element though their rows alternate; empty matrices share nothing."""
    base, stride = 1 << 20, 64
    cols = [_lib.tgs_matrix(base + 4 * 8 * k, 100, 8, stride, F32) for k in range(8)]
    rc, h = create(cols[:4] + [_lib.tgs_matrix(base, 0, 8, stride, F32)], cols[4:] + [_lib.tgs_matrix(base, 0, 8, 8, F16)])
    assert rc == 0
    assert _lib.load().tgs_gradient_clip_destroy(h) == 0
    wide = _lib.tgs_matrix(base + 4 * 8 * 3, 100, 9, stride, F32)   # a column into the next
    rc, _ = create(cols[:3] + [wide] + cols[4:5])
    assert rc == _lib.TGS_ERR_INVALID and "grads[4] overlaps grads[3]" in words()
    inner = _lib.tgs_matrix(base + 4 * (64 * 7 + 20), 1, 8, 8, F32)   # within a row of others
    rc, _ = create(cols + [inner])
    assert rc == _lib.TGS_ERR_INVALID and "grads[8] overlaps grads[" in words()


@pytest.mark.parametrize("number", [np.float32, np.float64, np.int64, torch.tensor, int], ids=str)
def test_numbers(number):
    """max_norm, scale and epsilon from NumPy and torch reach the library as the numbers that they are."""
    lib = _lib.load()
    rc, h = create([_lib.tgs_matrix(1 << 20, 4, 8, 8, F32)])
    assert rc == 0
    assert lib.tgs_gradient_clip_run(h, number(-1), number(1), number(0), None, None) == _lib.TGS_ERR_INVALID
    assert "max_norm -1" in words()
    assert lib.tgs_gradient_clip_run(h, number(1), number(-2), number(0), None, None) == _lib.TGS_ERR_INVALID
    assert "scale -2" in words()
    assert lib.tgs_gradient_clip_destroy(h) == 0

"""How a 4-bit linear layer's calls are taken, by sizes and types (host only):
the kernel and tile, and where results are stored past the caches."""
import ctypes

import pytest

from hi_amd import _lib

F32, BF16, MX4 = _lib.DTYPE_F32, _lib.DTYPE_BF16, _lib.DTYPE_MX4
FEW = (16, 64)


def path(rows, n, k, x_dtype=MX4, out_dtype=F32):
    """((rows, outputs) of a workgroup, stored past the caches)"""
    out = [ctypes.c_int(-1) for _ in range(3)]
    assert _lib.load().hi_rocm_debug_mx4_linear(rows, n, k, x_dtype, out_dtype, *map(ctypes.byref, out)) == 0
    return (out[0].value, out[1].value), bool(out[2].value)


@pytest.mark.parametrize("rows,n,out_dtype,past", [
    (128, 4096, BF16, False), (128, 4096, F32, False), (320, 4096, BF16, False),  # up to one L2
    (320, 4096, F32, True), (320, 16384, BF16, True), (2048, 4096, BF16, True),   # up to all eight
    (2048, 4096, F32, False), (1024, 16384, F32, False), (8192, 4096, F32, False), (6000, 16384, BF16, False),
    (8192, 16384, BF16, True), (8192, 16384, F32, True)])                         # past the last-level cache
def test_stores_past_the_caches(rows, n, out_dtype, past):
    """By the result's bytes: neither always nor never."""
    tile, got = path(rows, n, 4096, out_dtype=out_dtype)
    assert tile != FEW and got is past


def test_few_rows_are_stored_as_they_come():
    for rows in (1, 5, 16):
        assert path(rows, 151936, 4096, x_dtype=BF16) == (FEW, False)
    assert path(1, 1 << 24, 512, x_dtype=BF16) == (FEW, False)  # 67 MB


def test_refused():
    lib, i = _lib.load(), ctypes.byref(ctypes.c_int())
    good = [4, 64, 64, BF16, F32, i, i, i]
    assert lib.hi_rocm_debug_mx4_linear(*good) == _lib.OK
    for at, bad, status in ((0, 0, _lib.ERR_ARGS), (1, -1, _lib.ERR_ARGS), (2, 0, _lib.ERR_ARGS), (3, F32, _lib.ERR_ARGS),
                            (4, MX4, _lib.ERR_ARGS), (5, None, _lib.ERR_ARGS), (6, None, _lib.ERR_ARGS),
                            (7, None, _lib.ERR_ARGS), (2, 48, _lib.ERR_UNSUPPORTED), (0, (1 << 22) + 1, _lib.ERR_UNSUPPORTED),
                            (1, (1 << 24) + 1, _lib.ERR_UNSUPPORTED)):
        args = list(good)
        args[at] = bad
        assert lib.hi_rocm_debug_mx4_linear(*args) == status
        assert b"hi_rocm_debug_mx4_linear:" in lib.hi_rocm_last_error()

"""How a 4-bit linear layer's calls are taken, by sizes and types (host only):
the kernel and tile, and where results are stored past the caches."""
import ctypes

import pytest

from hi_amd import _lib

F32, BF16, MX4 = _lib.DTYPE_F32, _lib.DTYPE_BF16, _lib.DTYPE_MX4
FEW = (16, 64)

# Rows, outputs and inputs that no tile divides (the last tile of rows has one row, or one
# less than whole; a k that ends inside a quad or a step), and the way each is taken.
CASES = [
    (4093, 16385, 544, (128, 256)), (8190, 4097, 1184, (128, 256)), (4097, 16390, 160, (128, 256)),
    (2999, 9001, 1184, (96, 256)), (509, 16385, 544, (96, 256)), (1027, 8200, 160, (96, 256)),
    (130, 16400, 1184, (64, 256)), (1021, 4090, 4640, (64, 256)), (33, 70001, 544, (64, 256)),
    (1027, 8200, 4640, (64, 128)), (509, 16385, 1184, (64, 128)), (330, 4090, 4640, (64, 128)),
    (300, 2050, 544, (32, 256)), (600, 2050, 1184, (32, 256)), (500, 4001, 160, (32, 256)),
    (300, 2050, 4640, (32, 128)), (130, 4097, 1184, (32, 128)), (33, 9001, 4640, (32, 128)),
    (700, 700, 1184, (32, 64)), (190, 70, 4640, (32, 64)), (300, 1001, 8224, (32, 64)), (300, 1001, 1184, (32, 64)),
    (90, 1000, 544, FEW), (16, 333, 1184, FEW), (1, 70, 160, FEW)]
TILES = {(128, 256), (96, 256), (64, 256), (64, 128), (32, 256), (32, 128), (32, 64), FEW}


def path(rows, n, k, x_dtype=MX4, out_dtype=F32):
    """((rows, outputs) of a workgroup, stored past the caches)"""
    out = [ctypes.c_int(-1) for _ in range(3)]
    assert _lib.load().hi_rocm_debug_mx4_linear(rows, n, k, x_dtype, out_dtype, *map(ctypes.byref, out)) == 0
    return (out[0].value, out[1].value), bool(out[2].value)


def workspace(rows, n, k):
    """Bytes that a call with bf16 rows takes."""
    out = ctypes.c_size_t()
    assert _lib.load().hi_rocm_mx4_linear_workspace_bytes(rows, n, k, ctypes.byref(out)) == 0
    return out.value


@pytest.mark.parametrize("rows,n,k,tile", CASES)
def test_tile(rows, n, k, tile):
    assert path(rows, n, k)[0] == tile


def test_cases_cover_every_way():
    assert {c[3] for c in CASES} == TILES
    whole = [c for c in CASES if c[3] != FEW and (c[0] % c[3][0] == 0 or c[1] % c[3][1] == 0 or c[2] % 512 == 0)]
    assert not whole
    # more rows than 16 are rounded by the workgroups that multiply them, and beforehand
    ways = {path(rows, n, k, x_dtype=BF16)[0] == FEW for rows, n, k, tile in CASES if rows > 16 and tile != FEW}
    assert ways == {True, False}
    for rows, n, k, tile in CASES:
        assert (workspace(rows, n, k) == 0) == (path(rows, n, k, x_dtype=BF16)[0] == FEW)


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

"""Which tile the 8-bit products take, without a GPU: the sizes at the rules' borders."""

import ctypes

import pytest

from nanotitan_amd import capi

PLAIN, SWIGLU, GELU, GRADIENT = (capi.NT_INT8_PLAIN, capi.NT_INT8_SWIGLU, capi.NT_INT8_GELU,
                                 capi.NT_INT8_GRADIENT)


def tile(product, E, A, K, N, cus=256):
    rows, cols = ctypes.c_int32(-1), ctypes.c_int32(-1)
    st = capi.load().nt_int8_tile(product, E, A, K, N, cus, ctypes.byref(rows), ctypes.byref(cols))
    return (rows.value, cols.value) if st == capi.NT_OK else st


@pytest.mark.parametrize("product,E,A,K,N,want", [
    (PLAIN, 8, 192, 4096, 14336, (0, 0)), (PLAIN, 64, 64 * 24, 2048, 768, (0, 0)),
    (PLAIN, 1, 64, 4096, 4096, (0, 0)), (PLAIN, 1, 400, 4096, 4096, (128, 128)),
    (PLAIN, 8, 61440, 2048, 512, (128, 256)), (PLAIN, 8, 4000, 4096, 4096, (128, 128)),
    (GELU, 128, 14312, 2048, 768, (128, 128)), (SWIGLU, 8, 61440, 512, 2048, (128, 256)),
    (PLAIN, 8, 32768, 14336, 4096, (256, 256)), (PLAIN, 8, 32768, 8191, 4096, (128, 256)),
    (GELU, 8, 32768, 8192, 4096, (256, 256)), (SWIGLU, 8, 32768, 4096, 14336, (256, 256)),
    (SWIGLU, 8, 32768, 4095, 14336, (128, 256)),
    (GRADIENT, 8, 4188, 512, 2048, (128, 128)), (GRADIENT, 8, 871, 4096, 14336, (128, 128)),
    (GRADIENT, 8, 61440, 512, 2048, (128, 256)), (GRADIENT, 128, 14312, 768, 2048, (128, 256))])
def test_tiles_of_256_cus(product, E, A, K, N, want):
    assert tile(product, E, A, K, N) == want


def test_fewer_cus_take_wide_tiles_earlier():
    assert tile(PLAIN, 8, 4000, 4096, 4096, 64) == (128, 256)
    assert tile(GRADIENT, 8, 4188, 512, 2048, 64) == (128, 128)
    assert tile(GRADIENT, 8, 4188, 512, 2048, 32) == (128, 256)


def test_refusals():
    for args in ((-1, 1, 4, 8, 8), (4, 1, 4, 8, 8), (PLAIN, 0, 4, 8, 8), (PLAIN, 1, -1, 8, 8),
                 (PLAIN, 1, 4, 0, 8), (PLAIN, 1, 4, 8, 8, 0)):
        assert tile(*args) == capi.NT_ERR_INVALID_ARG
    assert tile(PLAIN, 1025, 4, 8, 8) == capi.NT_ERR_TOO_MANY_EXPERTS
    assert tile(PLAIN, 1, 2**24, 8, 8) == capi.NT_ERR_TOO_LARGE
    lib, n = capi.load(), ctypes.c_int32()
    assert lib.nt_int8_tile(PLAIN, 1, 4, 8, 8, 256, None, ctypes.byref(n)) \
        == lib.nt_int8_tile(PLAIN, 1, 4, 8, 8, 256, ctypes.byref(n), None) \
        == capi.NT_ERR_INVALID_ARG

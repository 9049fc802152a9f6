"""Terms of gradients of every type: sizes and refusals, without a GPU."""

import pytest

from nanotitan_amd import capi

F32, F64, F16, BF = capi.NT_F32, capi.NT_F64, capi.NT_F16, capi.NT_BF16
P = 4096  # a non-null, aligned address: none of these calls gets as far as using it
BAD = capi.NT_ERR_INVALID_ARG


@pytest.mark.parametrize("dtype", [F32, F16, BF])
def test_rows_terms_refuse(dtype):
    fn = capi.load().nt_int8_rows_terms
    good = [dtype, P, P, P, 2, 4, 9, P]
    for i, v, code in [(0, F64, capi.NT_ERR_DTYPE), (1, None, BAD), (2, None, BAD), (3, None, BAD),
                       (4, 0, BAD), (4, 1025, capi.NT_ERR_TOO_MANY_EXPERTS), (5, -1, BAD),
                       (5, 2**24, capi.NT_ERR_TOO_LARGE), (6, 0, BAD),
                       (6, 2**22 + 1, capi.NT_ERR_TOO_LARGE), (7, None, BAD), (7, P + 8, BAD)]:
        assert fn(*good[:i], v, *good[i + 1:], None) == code
    assert fn(dtype, None, None, None, 1, 0, 9, None, None) == capi.NT_OK


@pytest.mark.parametrize("dtype", [F32, F16, BF])
def test_products_of_terms_refuse(dtype):
    """A pitch of 0 says that dout is terms: N may be any number, scales are not needed."""
    lib = capi.load()
    sizes = [2, 4, 9, 15]
    for dout, scales, out, code in ((None, P, P, BAD), (P + 8, None, P, BAD), (P, P, None, BAD)):
        head = [dtype, P, scales, P, dout, 0]
        assert lib.nt_int8_grouped_gemm_dx(*head, *sizes, out, None) == code
        assert lib.nt_int8_grouped_gemm_dx_gelu(*head, P, P, *sizes, out, None) == code
        assert lib.nt_int8_grouped_gemm_dx_swiglu(*head, P, P, P, P, *sizes, out, P, None) == code
    assert lib.nt_int8_grouped_gemm_dx(dtype, P, P, P, P, 0, 2, 4, 9, 2**22 + 1, P,
                                       None) == capi.NT_ERR_TOO_LARGE
    if dtype != F32:
        assert lib.nt_int8_grouped_gemm_dx(dtype, P, None, P, P, 16, *sizes, P, None) == BAD

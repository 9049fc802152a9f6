"""8-bit checkpoints of more chunks than a launch has threads are refused by name."""

import pytest

from nanotitan_amd import capi

BF = capi.NT_BF16
P = 4096  # a non-null address: none of these calls gets as far as using it

# (fn, the arguments after rows and f, of which one is missing: an invalid argument, which
# is found after the sizes)
CALLS = [("nt_checkpoint8", lambda r, f: (BF, P, r, f, P, None, None)),
         ("nt_checkpoint8_decode", lambda r, f: (BF, P, P, r, f, None, None)),
         ("nt_gelu_checkpoint8", lambda r, f: (BF, P, r, f, None, P, P, None)),
         ("nt_gelu_backward8", lambda r, f: (BF, P, P, P, r, f, None, None, None)),
         ("nt_swiglu_checkpoint8", lambda r, f: (BF, P, P, r, f, None, P, P, P, P, None)),
         ("nt_swiglu_backward8", lambda r, f: (BF, P, P, P, P, P, r, f, None, P, None, None))]


@pytest.mark.parametrize("fn,args", CALLS, ids=[c[0] for c in CALLS])
def test_largest_sizes(fn, args):
    call = lambda r, f: getattr(capi.load(), fn)(*args(r, f))  # noqa: E731
    # two threads for 32 columns of a row, workgroups of 256, fewer than 2^32 in all
    assert call(2**27, 512) == capi.NT_ERR_TOO_LARGE  # 2^32 threads
    assert call(2**27 - 7, 512) == capi.NT_ERR_TOO_LARGE  # 2^32 - 224: workgroups up to 2^32
    assert call(2**27 - 8, 512) == capi.NT_ERR_INVALID_ARG  # 2^32 - 256
    assert call(2**31 - 1, 1) == capi.NT_ERR_TOO_LARGE  # 2^32 - 2
    assert call(2**31 - 128, 32) == capi.NT_ERR_INVALID_ARG  # 2^32 - 256

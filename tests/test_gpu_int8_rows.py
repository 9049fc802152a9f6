"""Rows and weights to 8-bit integers and back, against the definition in 64 bits: integers and
scales are equal, values are rounded once."""

import pytest
import torch

from nanotitan_amd.moe_ops import (
    Int8Weight,
    int8_rows,
    int8_rows_decode,
    int8_weight,
    int8_weight_decode,
)
from tests import int8_oracle as O

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _values(*shape, dtype, seed=0, shift=0):
    g = torch.Generator().manual_seed(seed)
    n = 1
    for s in shape:
        n *= s
    buf = torch.randn(n + shift, generator=g).to(dtype).cuda()
    return buf[shift:].view(*shape)  # any alignment that a view can have


def _check_rows(x):
    codes, scales = int8_rows(x)
    f = x.shape[1]
    q, s = O.held(x.cpu(), 1)
    assert codes.shape == (-(-x.shape[0] // 16), O.pitch(f) // 64, 4, 16, 16)
    assert codes.dtype == torch.int8
    plain = O.plain_rows(codes)[:x.shape[0]]
    assert torch.equal(plain[:, :f].cpu().long(), q)
    assert not bool(plain[:, f:].any())
    assert torch.equal(scales.cpu().nan_to_num(-1.0), s.view(-1).nan_to_num(-1.0))
    for dtype in {x.dtype, torch.float32}:
        got = int8_rows_decode(codes, scales, f, dtype)
        most = torch.finfo(dtype).max
        want = (q.float() * s).clamp(-most, most).to(dtype)  # one product in 32 bits, one rounding
        assert torch.equal(got.cpu().nan_to_num(-1.0), want.nan_to_num(-1.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,f", [(1, 1), (3, 15), (5, 128), (7, 300), (9, 1024), (2, 1025),
                                    (1500, 1365), (1030, 2048), (6, 2049), (4, 4096), (3, 4097),
                                    (2, 8192), (3, 14336), (2, 16384), (2, 16385), (1, 40001)])
def test_rows(dtype, rows, f):
    _check_rows(_values(rows, f, dtype=TYPES[dtype], seed=f))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_any_alignment(dtype):
    for shift in (1, 3, 5):
        _check_rows(_values(17, 333, dtype=TYPES[dtype], seed=shift, shift=shift))


@pytest.mark.parametrize("dtype", TYPES)
def test_half_way_values_go_to_the_even_integer(dtype):
    # a largest value of 127 2^j makes the scale 2^j: every half is a tie
    halves = torch.arange(-253, 254, 2).double() / 2
    for j in (-6, 0, 5):
        x = torch.cat([halves, torch.tensor([127.0, -127.0]).double()]) * 2.0**j
        _check_rows(x.to(TYPES[dtype]).view(1, -1).cuda())


def test_values_next_to_a_border():
    # the float32 neighbours of (k + 1/2) s for scales of every last bit
    g = torch.Generator().manual_seed(3)
    most = (torch.rand(64, generator=g) + 1.0) * 100.0
    s = (most.double() / 127.0).float()
    k = torch.arange(-126, 126).double() + 0.5
    at = (k.view(1, -1) * s.double().view(-1, 1)).float()
    up = torch.nextafter(at, torch.full_like(at, 1e30))
    down = torch.nextafter(at, torch.full_like(at, -1e30))
    _check_rows(torch.cat([most.view(-1, 1), at, up, down], 1).cuda())


@pytest.mark.parametrize("dtype", TYPES)
def test_extremes(dtype):
    t = TYPES[dtype]
    fi = torch.finfo(t)
    x = torch.zeros(9, 200, dtype=t)
    x[1, 5], x[1, 6] = fi.max, -fi.max / 3
    x[2, 7], x[2, 9] = fi.smallest_normal, -fi.smallest_normal / 2
    x[3, :] = fi.smallest_normal / 4  # subnormal
    x[4, 3], x[4, 4] = float("inf"), 1.0
    x[5, 199], x[5, 0] = float("nan"), 2.0
    x[6, 0], x[6, 1] = -float("inf"), float("nan")
    x[7, 100] = -0.0
    x[8, :] = -1.0
    _check_rows(x.cuda())


def test_no_rows():
    codes, scales = int8_rows(torch.zeros(0, 300, device="cuda"))
    assert codes.shape == (0, 6, 4, 16, 16) and scales.shape == (0,)
    assert int8_rows_decode(codes, scales, 300, torch.float16).shape == (0, 300)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,K,N", [(1, 1, 1), (2, 5, 3), (3, 64, 64), (2, 65, 130), (1, 128, 4),
                                   (2, 300, 1365), (5, 129, 63), (1, 1100, 257)])
def test_weights(dtype, E, K, N):
    W = _values(E, K, N, dtype=TYPES[dtype], seed=K, shift=1)
    _check_weight(W)


def _check_weight(W):
    E, K, N = W.shape
    w = int8_weight(W)
    q, s = O.held(W.cpu(), 1)
    assert w.shape == (E, K, N)
    assert torch.equal(w.codes.cpu(), O.blocks(q))
    assert torch.equal(w.scale.cpu().nan_to_num(-1.0), s.view(E, N).nan_to_num(-1.0))
    got = int8_weight_decode(w, W.dtype)
    most = torch.finfo(W.dtype).max
    want = (q.float() * s).clamp(-most, most).to(W.dtype)
    assert torch.equal(got.cpu().nan_to_num(-1.0), want.nan_to_num(-1.0))


def test_weights_with_channels_of_zeros_and_infinities():
    W = _values(2, 70, 70, dtype=torch.float32)
    W[0, :, 3] = 0.0
    W[1, 69, 4] = float("inf")
    W[0, 0, 69] = float("nan")
    W[1, :, 68] = 1e-42
    _check_weight(W)


def test_two_dimensions_are_one_expert():
    W = _values(40, 70, dtype=torch.bfloat16)
    a, b = int8_weight(W), int8_weight(W.unsqueeze(0))
    assert a.shape == b.shape == (1, 40, 70) and torch.equal(a.codes, b.codes)


def test_past_32_bit_offsets():
    """The last rows of 2^31 values, and the last expert of weights of 2^32 integers."""
    A, f = 2**21 + 5, 1024
    x = torch.zeros(A, f, dtype=torch.float16, device="cuda")
    tail = _values(7, f, dtype=torch.float16)
    x[-7:] = tail
    codes, scales = int8_rows(x)
    c, s = int8_rows(tail)
    last = O.plain_rows(codes[-2:])[:16 + A % 16]
    assert torch.equal(last[-7:], O.plain_rows(c)[:7]) and torch.equal(scales[-7:], s)
    assert not bool(last[:-7].any())
    back = int8_rows_decode(codes, scales, f, torch.float16)
    assert torch.equal(back[-7:], int8_rows_decode(c, s, f, torch.float16))
    del x, codes, back
    W = torch.zeros(33, 8192, 16384, dtype=torch.bfloat16, device="cuda")
    W[32, -70:, -70:] = _values(70, 70, dtype=torch.bfloat16)
    w = int8_weight(W)
    one = int8_weight(W[32])
    assert torch.equal(w.codes[32], one.codes[0]) and torch.equal(w.scale[32], one.scale[0])
    assert not bool(w.codes[31].any())
    last = int8_weight_decode(w, torch.bfloat16)[32]
    assert torch.equal(last, int8_weight_decode(one, torch.bfloat16)[0])


def test_refusals():
    x = torch.zeros(4, 64, device="cuda")
    codes, scales = int8_rows(x)
    for bad in (lambda: int8_rows(x.double()), lambda: int8_rows(x.view(-1)),
                lambda: int8_rows_decode(codes, scales, 200, torch.float32),
                lambda: int8_rows_decode(codes, scales.repeat(5), 64, torch.float32),
                lambda: int8_rows_decode(codes.float(), scales, 64, torch.float32),
                lambda: int8_rows_decode(codes, scales, 64, torch.float64),
                lambda: int8_weight(x.double()), lambda: int8_weight(x.view(-1)),
                lambda: int8_weight(torch.zeros(0, 4, 4, device="cuda")),
                lambda: int8_weight(torch.zeros(1, 2**17 + 1, 1, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()
    w = int8_weight(x)
    with pytest.raises(RuntimeError, match="integers"):
        int8_weight_decode(Int8Weight(w.codes[:, :, :1].contiguous(), w.scale, w.shape),
                           torch.float32)

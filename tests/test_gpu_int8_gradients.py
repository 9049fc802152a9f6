"""Gradients through 8-bit weights at the ends of their types: infinities, NaN, the largest values."""

import pytest
import torch

from nanotitan_amd import moe_ops
from nanotitan_amd.moe_ops import (
    int8_gelu_ffn_fn,
    int8_grouped_gemm_fn,
    int8_swiglu_ffn_fn,
    int8_weight,
)

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _positive(*shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return ((torch.rand(*shape, generator=g) + 0.5) * scale).cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("op", ["product", "gelu", "swiglu"])
def test_infinite_gradients_stay_infinite(dtype, op, monkeypatch):
    """With positive tokens and weights every factor on the way is positive: a row with an
    infinity is that infinity, one with a NaN is NaN, the others are as without."""
    monkeypatch.setattr(moe_ops, "_int8_direct", lambda d, E, K: True)
    t, A, d, f = TYPES[dtype], 11, 70, 90
    up = [int8_weight(_positive(d, f, seed=i, scale=1 / d)) for i in (1, 2)]
    down = int8_weight(_positive(f, d, seed=3, scale=1 / f))
    fn = {"product": lambda v: int8_grouped_gemm_fn(v, up[0]),
          "gelu": lambda v: int8_gelu_ffn_fn(v, up[0], down),
          "swiglu": lambda v: int8_swiglu_ffn_fn(v, *up, down)}[op]
    x = _positive(A, d, seed=4).to(t).requires_grad_()
    y = fn(x)
    dy = _positive(*y.shape, seed=5).to(t)
    want, = torch.autograd.grad(y, x, dy, retain_graph=True)
    assert bool(want.isfinite().all())
    dy[1, 3], dy[4, 0], dy[6, 5] = float("inf"), -float("inf"), float("nan")
    got, = torch.autograd.grad(y, x, dy)
    assert bool((got[1] == float("inf")).all()) and bool((got[4] == -float("inf")).all())
    assert bool(got[6].isnan().all())
    keep = [i for i in range(A) if i not in (1, 4, 6)]
    assert torch.equal(got[keep], want[keep])


def test_the_largest_float32_gradient(monkeypatch):
    """A value that bfloat16 would round to an infinity: its terms are finite."""
    monkeypatch.setattr(moe_ops, "_int8_direct", lambda d, E, K: True)
    w = int8_weight(torch.tensor([[127.0], [1.0], [-1.0]], device="cuda"))  # scale 1
    x = torch.ones(2, 3, device="cuda", requires_grad=True)
    dout = torch.tensor([[3.4e38], [-3.4e38]], device="cuda")
    got, = torch.autograd.grad(int8_grouped_gemm_fn(x, w), x, dout)
    assert got[:, 0].tolist() == [float("inf"), -float("inf")]
    # three terms hold 2^-25 of the value, their sum rounds once more
    assert bool(((got[:, 1] - dout[:, 0]).abs() <= 2.0**-23 * 3.4e38).all())
    assert torch.equal(got[:, 2], -got[:, 1])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("A", [80, 6000])  # tiles of 128 and of 256 columns
def test_the_direct_product_takes_the_weights_as_decoded(dtype, A):
    """Rows of one 1 pick the weights out: rounded once to 16 bits, past the type's largest that,
    a NaN channel NaN, as ``int8_weight_decode`` gives them."""
    t, K, N = TYPES[dtype], 1500, 80
    g = torch.Generator().manual_seed(1)
    W = torch.randn(1, K, N, generator=g)
    most = torch.finfo(t).max
    W[0, :, 3] *= 1e-6
    for n, big in ((10, 1.0), (11, 0.99), (33, 1.5)):
        W[0, 7 + n, n] = big * most if n != 33 or t == torch.float16 else 3.4e38
    W[0, 5, 70] = float("nan")
    w = int8_weight(W.cuda())
    off = torch.tensor([0, A], dtype=torch.int32, device="cuda")
    dout = torch.zeros(A, N, dtype=t)
    dout[torch.arange(A), torch.arange(A) % N] = 1.0
    held = moe_ops.int8_weight_decode(w, t)[0].t()
    ext = moe_ops.get_hip_extension()
    got = ext.int8_dx(dout.cuda(), off, w.codes, w.scale, K)
    # 0 * NaN: with the NaN channel every row is NaN; without it the rows are the weights
    assert bool(got.isnan().all())
    scale = w.scale.clone()
    scale[0, 70] = 1.0
    got = ext.int8_dx(dout.cuda(), off, w.codes, scale, K)
    want = held.clone()
    want[70] = 0.0  # (its integers are 0)
    assert torch.equal(got, want.repeat(-(-A // N), 1)[:A])

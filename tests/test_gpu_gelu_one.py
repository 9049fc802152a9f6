"""One GELU for the experts: the 8-bit path, the few-token layer and the plain FFN
agree, and stay relatively exact where the normal distribution's tail is small."""

import math
from types import SimpleNamespace

import pytest
import torch

import tests.test_gpu_moe_block as blocks
from nanotitan_amd import moe_ops
from nanotitan_amd.layer import MoEBlock
from tests.test_block_ops_cpu import held64

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0**-24


def _cdf64(x):
    return 0.5 * torch.special.erfc(-x * 0.5**0.5)


def _slope64(x):
    return _cdf64(x) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


def _fit(x):
    """Relative error of a 16-bit GELU of float32 steps: the fit's 1.2e-7 = 2 U, 8 roundings, and
    exp2's argument: x^2 / 2 in natural units, rounded at six places (the constant of |x| /
    sqrt(2) and its product, each squared, the square and its product with log2 e)."""
    return (10 + 6 * 0.5 * x * x) * U


def _tail_tolerance(x, want, dtype):
    eps = torch.finfo(dtype).eps
    if dtype == torch.float32:
        # 0.5 (1 + erf): erf within two units of one at 1, and cancelled there
        return 8 * U * x.abs()
    # half a step of the subnormals: fp16 2^-14 2^-10 / 2, bf16 2^-126 2^-7 / 2
    sub = 2.0**-25 if dtype == torch.float16 else 2.0**-134
    return (eps / 2 + _fit(x)) * want.abs() * (1 + eps) + sub


def _every_value(dtype):
    """All finite values of a 16-bit type, or a fine grid, with |x| < 13, in rows of 32 columns."""
    if dtype == torch.float32:
        return torch.linspace(-13, 13, 32 * 2048).view(-1, 32)
    x = torch.arange(-2**15, 2**15, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[x.float().abs() < 13]
    return torch.cat([x, x.new_zeros(-len(x) % 32)]).view(-1, 32)


@pytest.mark.parametrize("dtype", TYPES)
def test_gelu8_of_every_value(ext, dtype):
    x = _every_value(TYPES[dtype])
    got = moe_ops.gelu8_fn(x.cuda()).cpu().double()
    x64 = x.double()
    want = x64 * _cdf64(x64)
    off = (got - want).abs() - _tail_tolerance(x64, want, x.dtype)
    assert bool((off <= 0).all()), float(x64.flatten()[off.flatten().argmax()])


@pytest.mark.parametrize("dtype", TYPES)
def test_gelu8_slope_in_the_tail(ext, dtype):
    """Blocks of one value, which 8 bits hold to within 1/127.5: gelu' and gelu of the value kept."""
    dt = TYPES[dtype]
    x = torch.linspace(-12, 12, 997).to(dt).view(-1, 1).expand(-1, 32).contiguous()
    codes, exps = moe_ops.checkpoint8(x.cuda())
    d = torch.ones_like(x).cuda()
    dh, act = ext.gelu_backward8(d, codes, exps, True)
    k64 = held64(x.double())
    want = k64 * _cdf64(k64)
    off = (act.cpu().double() - want).abs() - _tail_tolerance(k64, want, dt)
    assert bool((off <= 0).all()), float(k64.flatten()[off.flatten().argmax()])
    # the slope's two terms cancel at -0.75 only; in the tail x phi(x) outweighs Phi(x) x^2 times
    size = _cdf64(k64) + k64.abs() * torch.exp(-0.5 * k64 * k64) / math.sqrt(2 * math.pi)
    want = _slope64(k64)
    if dt == torch.float32:
        tol = 16 * U * (1 + k64.abs())
    else:
        tol = torch.finfo(dt).eps / 2 * want.abs() + _fit(k64) * size + (
            2.0**-25 if dt == torch.float16 else 2.0**-134)
    off = (dh.cpu().double() - want).abs() - tol
    assert bool((off <= 0).all()), float(k64.flatten()[off.flatten().argmax()])


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T", [12, 40])
def test_few_tokens_in_the_tail(ext, dtype, T):
    """One expert whose projections are diagonal: the output is the rounded hidden row."""
    dt = TYPES[dtype]
    n = 256
    z = torch.linspace(-12, -3, n).to(dt)
    up, down = torch.diag(z).unsqueeze(0).cuda(), torch.eye(n, dtype=dt).unsqueeze(0).cuda()
    x = torch.ones(T, n, dtype=dt, device="cuda")
    with torch.no_grad():
        got = moe_ops.moe_few_tokens(x, (up, down), 1, logits=torch.zeros(T, 1, device="cuda"))[0]
    z64 = z.double()
    want = z64 * _cdf64(z64)
    off = (got.cpu().double() - want).abs() - _tail_tolerance(z64, want, dt)
    assert bool((off <= 0).all()), float(z64[off.max(0).values.argmax()])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,f", [(128, 256), (512, 2048)])
def test_checkpoints_leave_gelu_experts_forward_alone(ext, dtype, d, f):
    """The same bits with and without 8-bit checkpoints, and in training and evaluation."""
    dt = TYPES[dtype]

    def block(**over):
        cfg = dict(num_experts=8, top_k=2, d_model=d, ffn_in=f, dtype=dt, moe_backend="hip",
                   moe_router_dtype=torch.float32, router_alpha=0.01)
        torch.manual_seed(0)
        with torch.device("cuda"):
            return MoEBlock(SimpleNamespace(**cfg | over), norm="layer", ffn="gelu")

    plain, kept = block(), block(ffn_checkpoint8=True)
    kept.load_state_dict(plain.state_dict())
    with torch.no_grad():  # pre-activations of a few deviations: tails too
        for b in (plain, kept):
            b.moe.experts.W_up.copy_(torch.randn(b.moe.experts.W_up.shape, generator=torch.
                                                 Generator().manual_seed(1)) * 2 * d**-0.5)
    x = torch.randn(4, 100, d, device="cuda").to(dt)
    out = plain(x)[0]
    assert torch.equal(kept(x)[0], out)
    with torch.no_grad():
        assert torch.equal(kept(x)[0], out)


def test_checkpoints_change_gelu_experts_gradients_by_their_rounding(ext):
    """The blocks' test of outputs and weight gradients, with GELU experts."""
    blocks.test_checkpoints_change_the_weight_gradients_by_their_rounding(ext, blocks.KINDS[2])


@pytest.mark.parametrize("fn", ["swiglu", "gelu"])
def test_ffn8_without_rows(ext, fn):
    """No row, and experts of which none has one: gradients of zero."""
    d, f, E = 64, 96, 3
    up = [torch.randn(E, d, f, device="cuda", requires_grad=True)
          for _ in range(2 if fn == "swiglu" else 1)]
    down = torch.randn(E, f, d, device="cuda", requires_grad=True)
    X = torch.randn(0, d, device="cuda", requires_grad=True)
    off = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    call = moe_ops.swiglu_ffn8_fn if fn == "swiglu" else moe_ops.grouped_gelu_ffn8_fn
    y = call(X, *up, down, off)
    assert y.shape == (0, d)
    dX, *dW = torch.autograd.grad(y, [X, *up, down], torch.zeros_like(y))
    assert dX.shape == (0, d) and all(float(w.abs().max()) == 0.0 for w in dW)

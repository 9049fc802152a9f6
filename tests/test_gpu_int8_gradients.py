"""Gradients through 8-bit weights: at the ends of their types (infinities, NaN, the largest and
smallest values), of the weights held exactly, and of weights rounded to 16 bits where a caller
asks for that."""

from types import SimpleNamespace

import pytest
import torch

from nanotitan_amd import moe_ops
from nanotitan_amd.layer import GeluExpertFFN, Int8ExpertFFN, ModelShardSpec
from nanotitan_amd.moe_ops import (
    int8_gelu_ffn_fn,
    int8_grouped_gemm_fn,
    int8_swiglu_ffn_fn,
    int8_weight,
    int8_weight_decode,
)

pytestmark = pytest.mark.gpu

U = 2.0**-24
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
    held = int8_weight_decode(w, t)[0].t()
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


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_gradients_as_small_as_the_terms_hold(dtype, monkeypatch):
    """Products of gradient and scale of about 2^-100, each picked out by a row of one value."""
    monkeypatch.setattr(moe_ops, "_int8_direct", lambda d, E, K: True)
    t, K, N = TYPES[dtype], 100, 64
    g = torch.Generator().manual_seed(1)
    W = torch.randn(K, N, generator=g) * 2.0**-58  # scales of about 2^-64
    w = int8_weight(W.cuda())
    v = (torch.rand(N, generator=g) + 1.0) * 2.0**-36
    dout = torch.diag(v.to(t)).cuda()
    x = torch.zeros(N, K, dtype=t, device="cuda", requires_grad=True)
    got, = torch.autograd.grad(int8_grouped_gemm_fn(x, w), x, dout)
    held = int8_weight_decode(w, torch.float32)[0].double().t()
    want = held * dout.double().sum(1, keepdim=True)
    # the terms, and the roundings of dout s, of q s and of the sum; of bfloat16 the output's:
    # 8 significant bits, so half of its last one is 2^-8 of the smallest value with that step
    half = torch.finfo(t).eps / 2
    rel = 2.0**-17 + half + 4 * U if t == torch.bfloat16 else 2.0**-25 + 6 * U
    assert bool(((got.double() - want).abs() <= rel * want.abs()).all())


# Rows an expert, and the widths: tiles of 128 columns, and of 256 with more than one a workgroup.
SIZES = {"few": ([3, 0, 16, 1], 300, 265), "odd": ([200, 0, 3, 50], 77, 130),
         "tiles": ([128, 129, 0, 300], 130, 72), "many": ([900, 0, 2500, 2600], 3001, 90)}


def _case(t, size, ends=False, seed=0):
    """(x, w, dout, offsets, their tensor): with ends, channels beyond float16 at both its ends."""
    counts, K, N = SIZES[size]
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    W = rand(len(counts), K, N) * K**-0.5
    dout = rand(off[-1], N)
    if ends:
        W[:, :, 3] *= 1e6
        W[:, :, 5] *= 1e-9
        dout[:, 3] *= 1e-3
        dout[::2, 3] = 0.0  # rows that the large channel does not drown
    x = rand(off[-1], K)
    return (x.to(t), int8_weight(W), dout.to(t), off,
            torch.tensor(off, dtype=torch.int32, device="cuda"))


def _rows(off):
    """Rows at the ends of the experts and in between, and their experts."""
    out = []
    for e, (a, b) in enumerate(zip(off, off[1:])):
        out += [(r, e) for r in sorted({*range(a, min(a + 9, b)), *range(max(a, b - 9), b),
                                        *range(a, b, 97)})]
    return [r for r, _ in out], [e for _, e in out]


def _product64(dout, w, rows, owners):
    """(dOut W^T, |dOut| |W|^T) in float64 for these rows, of the weights q s."""
    held = int8_weight_decode(w, torch.float32).cpu()
    d = dout.cpu().double()[rows]
    want = torch.stack([held[e].double() @ v for e, v in zip(owners, d)])
    size = torch.stack([held[e].double().abs() @ v.abs() for e, v in zip(owners, d)])
    return want, size


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("ends", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_product_gradient_is_of_the_weights_held(dtype, size, ends):
    t = TYPES[dtype]
    x, w, dout, off, gpu_off = _case(t, size, ends)
    x.requires_grad_()
    got, = torch.autograd.grad(int8_grouped_gemm_fn(x, w, gpu_off), x, dout)
    rows, owners = _rows(off)
    want, size = _product64(dout, w, rows, owners)
    # q s and dOut s to float32, the two terms, a float32 sum of 2 N products, one rounding
    N, fi = dout.shape[1], torch.finfo(t)
    tol = (2.0**-17 + (2 * N + 3) * U) * size + fi.eps / 2 * want.abs() + fi.smallest_normal * fi.eps
    got = got.cpu().double()[rows]
    over = want.abs() > fi.max * (1 - fi.eps)  # past the type
    assert bool((((got - want).abs() <= tol) | over).all())
    assert ends or not bool(over.any())


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("ends", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_hidden_gradient_is_of_the_weights_held(dtype, size, ends):
    """The first product of a block's backward, elementwise, as the terms that it writes."""
    t = TYPES[dtype]
    _, w, dout, off, gpu_off = _case(t, size, ends)
    A, K, E = off[-1], w.shape[1], len(off) - 1
    g = torch.Generator(device="cuda").manual_seed(9)
    kept = [torch.randn(A, K, generator=g, device="cuda") for _ in range(2)]
    scales = [torch.rand(E, K, generator=g, device="cuda") + 0.01 for _ in range(2)]
    ext = moe_ops.get_hip_extension()
    gelu = ext.int8_dx_gelu(dout, kept[0], gpu_off, w.codes, w.scale, scales[0], K, True)
    gate, value = ext.int8_dx_swiglu(dout, *kept, gpu_off, w.codes, w.scale, *scales, K, True)
    rows, owners = _rows(off)
    d, size = _product64(dout, w, rows, owners)
    N = dout.shape[1]
    z, v = [k.cpu().double()[rows] for k in kept]
    s0, s1 = [s.cpu().double()[owners] for s in scales]
    sg = torch.sigmoid(z)
    # as of the product; then the operations on it, the hardware's exponential and reciprocal,
    # and the terms written (and of SwiGLU's slope 1 + z (1 - sg) where it cancels)
    rel = 2 * 2.0**-17 + (2 * N + 30) * U
    for got, f in ((gelu, z * s0), (gate, v * sg * (1 + z * (1 - sg)) * s0), (value, z * sg * s1)):
        sums = got[:, rows, :K].cpu().double().sum(0)
        tol = rel * size * f.abs() + 24 * U * size * (v * s0).abs() * (1 + z.abs()) + 2.0**-100
        err = (sums - d * f).abs() - tol
        assert bool((err <= 0).all()), float(err.max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
def test_block_gradient_is_its_stages(dtype, ffn):
    t = TYPES[dtype]
    x, up, _, off, gpu_off = _case(t, "odd", seed=1)
    d, f = up.shape[1:]
    val = _case(t, "odd", seed=2)[1]
    g = torch.Generator(device="cuda").manual_seed(3)
    down = int8_weight(torch.randn(len(off) - 1, f, d, generator=g, device="cuda") * f**-0.5)
    dy = torch.randn(off[-1], d, generator=g, device="cuda").to(t)
    x.requires_grad_()
    ups = (up, val) if ffn == "swiglu" else (up,)
    block = int8_swiglu_ffn_fn if ffn == "swiglu" else int8_gelu_ffn_fn
    ext = moe_ops.get_hip_extension()
    held = [h for w in (*ups, down) for h in (w.codes, w.scale)]
    for exact in (True, False):
        got, = torch.autograd.grad(block(x, *ups, down, gpu_off, exact_gradient=exact), x, dy)
        dout = dy if exact else moe_ops._aligned(dy)
        if ffn == "swiglu":
            _, *kept = ext.int8_swiglu_ffn(x.detach(), gpu_off, *held, True)
            terms = ext.int8_dx_swiglu(dout, *kept, gpu_off, down.codes, down.scale, up.scale,
                                       val.scale, f, exact)
            want = ext.int8_dx_terms(*terms, gpu_off, up.codes, up.scale, val.codes, d, t)
        else:
            _, slope = ext.int8_gelu_ffn(x.detach(), gpu_off, *held, True)
            terms = ext.int8_dx_gelu(dout, slope, gpu_off, down.codes, down.scale, up.scale, f,
                                     exact)
            want = ext.int8_dx_terms(terms, None, gpu_off, up.codes, up.scale, None, d, t)
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("direct", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_rounded_weights_by_choice(dtype, size, direct, monkeypatch):
    """exact_gradient=False: the weights in 16 bits, by either kernel; float32 has no such choice."""
    monkeypatch.setattr(moe_ops, "_int8_direct", lambda d, E, K: direct)
    t = TYPES[dtype]
    x, w, dout, off, gpu_off = _case(t, size)
    x.requires_grad_()
    got, = torch.autograd.grad(int8_grouped_gemm_fn(x, w, gpu_off, exact_gradient=False), x, dout)
    rows, owners = _rows(off)
    want, bound = _product64(dout, w, rows, owners)
    half = torch.finfo(t).eps / 2
    tol = (half + dout.shape[1] * U) * bound + half * want.abs()
    assert bool(((got.cpu().double()[rows] - want).abs() <= tol).all())
    x32 = x.detach().float().requires_grad_()
    y = int8_grouped_gemm_fn(x32, w, gpu_off, exact_gradient=False)
    a, = torch.autograd.grad(y, x32, dout.float())
    b, = torch.autograd.grad(int8_grouped_gemm_fn(x32, w, gpu_off), x32, dout.float())
    assert torch.equal(a, b)


def test_functions_without_the_choice_are_exact():
    x, w, dout, off, gpu_off = _case(torch.bfloat16, "odd")
    x.requires_grad_()
    want, = torch.autograd.grad(int8_grouped_gemm_fn(x, w, gpu_off), x, dout)
    got, = torch.autograd.grad(moe_ops.Int8GroupedGEMM_FN.apply(x, gpu_off, w), x, dout)
    assert torch.equal(got, want)


def test_the_module_takes_the_choice():
    cfg = SimpleNamespace(d_model=64, ffn_in=96, dtype=torch.bfloat16)
    with torch.device("cuda"):
        full = GeluExpertFFN(cfg, ModelShardSpec(per_rank_expert=2, end_expert_id=2), std=0.2)
    e = Int8ExpertFFN(full)
    off = torch.tensor([0, 30, 70], dtype=torch.int32, device="cuda")
    x = torch.randn(70, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn_like(x)
    grads = {}
    for exact in (True, False):
        cfg.int8_exact_gradient = exact
        grads[exact], = torch.autograd.grad(e(x, off), x, dy)
        want, = torch.autograd.grad(
            int8_gelu_ffn_fn(x, *e.weights(), off, exact_gradient=exact), x, dy)
        assert torch.equal(grads[exact], want)
    assert not torch.equal(grads[True], grads[False])
    del cfg.int8_exact_gradient
    assert torch.equal(torch.autograd.grad(e(x, off), x, dy)[0], grads[True])

"""8-bit activation checkpoints: the codes are exact (a power-of-two scale
rounds nothing but the value itself), and the activations' gradients are the
formula's at the values kept."""

import numpy as np
import pytest
import torch

from nanotitan_amd import moe_ops
from tests.test_block_ops_cpu import held64, kept64

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _rows(A, f, dtype, seed, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(A, f, generator=g)
    if spread:  # block sizes over many powers of two
        x = x * torch.exp2(torch.randint(-12, 12, (A, 1), generator=g).float())
    return x.to(dtype)


def _near(got, want, dtype, mag, ulps):
    """Half a step of the type, and `ulps` float32 roundings of values of size `mag`."""
    got = got.detach().cpu().double()
    tol = torch.finfo(dtype).eps / 2 * want.abs() + ulps * 2.0**-24 * mag
    if dtype == torch.float16:
        tol = tol + 2.0**-25  # half a step of its subnormals
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() - tol).max())


SHAPES = [(0, 64), (1, 1), (3, 7), (5, 31), (2, 32), (7, 33), (4, 100), (130, 1365), (257, 768)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("A,f", SHAPES)
def test_codes_and_values_are_exact(ext, dtype, A, f):
    x = _rows(A, f, TYPES[dtype], 1)
    codes, exps = moe_ops.checkpoint8(x.cuda())
    assert codes.dtype == torch.int8 and exps.dtype == torch.uint8
    want_codes, want_exps = kept64(x.double())
    assert torch.equal(codes.cpu(), want_codes) and torch.equal(exps.cpu(), want_exps)
    back = moe_ops.checkpoint8_decode(codes, exps, TYPES[dtype]).cpu()
    assert torch.equal(back.double(), held64(x.double()))


def test_borders_of_the_shared_power(ext):
    """Maxima around 127.5 units, halves that tie, subnormals, signed zeros, the largest values."""
    rows = []
    for top in (127.0, 127.49999, 127.5, 127.50001, 128.0, 64.0, 63.999996, 1.0):
        for p in (-120, -20, 0, 20, 119):
            rows.append([top * 2.0**p, 0.5 * 2.0**p, 1.5 * 2.0**p, -2.5 * 2.0**p])
    rows += [[0.0, -0.0, 0.0, 0.0], [1e-45, 0, 0, 0], [2.0**-126, 2.0**-127, -2.0**-130, 0],
             [3.4028235e38, -3.4028235e38, 1.0, 0]]
    x = torch.tensor(rows, dtype=torch.float32)
    codes, exps = moe_ops.checkpoint8(x.cuda())
    want_codes, want_exps = kept64(x.double())
    assert torch.equal(exps.cpu(), want_exps) and torch.equal(codes.cpu(), want_codes)
    back = moe_ops.checkpoint8_decode(codes, exps, torch.float32).cpu()
    assert torch.equal(back.double(), held64(x.double()))
    for dt in (torch.float16, torch.bfloat16):  # the largest values round up out of range
        most = torch.finfo(dt).max
        x = torch.tensor([[most, -most, most / 2, 1.0], [most * 0.99, 0, 0, 0]]).to(dt)
        back = moe_ops.checkpoint8_decode(*moe_ops.checkpoint8(x.cuda()), dt).cpu()
        assert torch.equal(back.double(), held64(x.double(), dt))
        assert float(back[0, 0]) == most and float(back[0, 1]) == -most


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_block_that_is_not_finite_decodes_to_nan(ext, bad):
    x = torch.randn(3, 96)
    x[1, 40] = bad
    codes, exps = moe_ops.checkpoint8(x.cuda())
    assert int(exps[1, 1]) == 255 and int(codes[1, 32:64].abs().sum()) == 0
    back = moe_ops.checkpoint8_decode(codes, exps, torch.float32).cpu()
    nan = torch.zeros(3, 96, dtype=torch.bool)
    nan[1, 32:64] = True
    assert torch.equal(back.isnan(), nan)
    leaf = x.cuda().requires_grad_()
    (dx,) = torch.autograd.grad(moe_ops.gelu8_fn(leaf), leaf, torch.ones_like(leaf))
    assert torch.equal(dx.cpu().isnan(), nan)


def _gelu64(h):
    return 0.5 * h * (1.0 + torch.erf(h * 0.5**0.5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("A,f", [(1, 1), (3, 7), (4, 100), (130, 1365)])
def test_gelu8(ext, dtype, A, f):
    dt = TYPES[dtype]
    x, d = _rows(A, f, dt, 2, spread=False) * 3, _rows(A, f, dt, 3, spread=False)
    h = x.cuda().requires_grad_()
    act = moe_ops.gelu8_fn(h)
    (dh,) = torch.autograd.grad(act, h, d.cuda())
    x64, d64 = x.double(), d.double()
    # erf and exp of float32: a few roundings each of |h| and of the slope
    _near(act, _gelu64(x64), dt, x64.abs(), 8)
    at = held64(x64).requires_grad_()
    (want,) = torch.autograd.grad(_gelu64(at), at, d64)
    _near(dh, want, dt, d64.abs() * (2 + x64.abs()), 16)
    with torch.no_grad():
        assert torch.equal(moe_ops.gelu8_fn(h), act)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("A,f", [(1, 1), (3, 7), (4, 100), (130, 1365)])
def test_swiglu8(ext, dtype, A, f):
    dt = TYPES[dtype]
    x, v = _rows(A, f, dt, 4, spread=False) * 4, _rows(A, f, dt, 5, spread=False)
    d = _rows(A, f, dt, 6, spread=False)
    g, val = x.cuda().requires_grad_(), v.cuda().requires_grad_()
    hidden = moe_ops.swiglu8_fn(g, val)
    dg, dv = torch.autograd.grad(hidden, [g, val], d.cuda())
    x64, v64, d64 = x.double(), v.double(), d.double()
    silu = torch.nn.functional.silu
    # exp2 of x log2(e): |x| roundings of its argument, then a reciprocal and three products
    _near(hidden, silu(x64) * v64, dt, (x64 * v64).abs() * (1 + x64.abs()), 8)
    a, b = held64(x64).requires_grad_(), held64(v64).requires_grad_()
    want_g, want_v = torch.autograd.grad(silu(a) * b, [a, b], d64)
    size = d64.abs() * (1 + x64.abs()) ** 2
    _near(dg, want_g, dt, size * (v64.abs() + 1), 16)
    _near(dv, want_v, dt, size, 16)
    with torch.no_grad():
        assert torch.equal(moe_ops.swiglu8_fn(g, val), hidden)


def test_gradients_against_differences(ext):
    """At inputs that 8 bits hold exactly the checkpoint changes nothing: central differences."""
    g = torch.Generator().manual_seed(7)
    # 2^-5 multiples below 127 / 32, with the largest value fixing the power
    x = torch.randint(-60, 61, (4, 64), generator=g).float() / 32
    v = torch.randint(-60, 61, (4, 64), generator=g).float() / 32
    x[:, ::32] = v[:, ::32] = 127 / 32
    d = torch.randn(4, 64, generator=g)
    a, b = x.cuda().requires_grad_(), v.cuda().requires_grad_()
    da, db = torch.autograd.grad(moe_ops.swiglu8_fn(a, b), [a, b], d.cuda())
    (dh,) = torch.autograd.grad(moe_ops.gelu8_fn(a), a, d.cuda())
    eps = 1e-5
    silu = torch.nn.functional.silu
    x64, v64, d64 = x.double(), v.double(), d.double()
    # central differences: eps^2 / 6 of the third derivative (below 2), and 2^-52 / eps
    tol = dict(rtol=2e-6, atol=2e-6)
    torch.testing.assert_close(
        da.cpu().double(), d64 * v64 * (silu(x64 + eps) - silu(x64 - eps)) / (2 * eps), **tol)
    torch.testing.assert_close(db.cpu().double(), d64 * silu(x64), **tol)
    torch.testing.assert_close(
        dh.cpu().double(), d64 * (_gelu64(x64 + eps) - _gelu64(x64 - eps)) / (2 * eps), **tol)


def test_rows_at_any_address_and_layout(ext):
    buf = torch.randn(1 + 37 * 77).to(torch.bfloat16).cuda()
    x = buf[1:].view(37, 77)
    codes, exps = moe_ops.checkpoint8(x)
    want_codes, want_exps = kept64(x.cpu().double())
    assert torch.equal(codes.cpu(), want_codes) and torch.equal(exps.cpu(), want_exps)
    t = torch.randn(64, 40).cuda().t().requires_grad_()  # not contiguous
    out = moe_ops.gelu8_fn(t)
    (dt,) = torch.autograd.grad(out, t, torch.ones(1, device="cuda").expand(40, 64))
    c = t.detach().contiguous().requires_grad_()
    out_c = moe_ops.gelu8_fn(c)
    assert torch.equal(out, out_c)
    assert torch.equal(dt, torch.autograd.grad(out_c, c, torch.ones_like(c))[0])


def test_in_a_graph_and_on_another_stream(ext):
    x = torch.randn(100, 200, device="cuda").requires_grad_()
    v = torch.randn(100, 200, device="cuda").requires_grad_()
    d = torch.randn(100, 200, device="cuda")

    def step():
        out = moe_ops.swiglu8_fn(x, v)
        # no eager graph of the leaves may live while one is captured
        return [out.detach(), *torch.autograd.grad(out, [x, v], d)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(on_side, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3):
        with torch.no_grad():
            x.copy_(torch.randn(100, 200, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip([t.clone() for t in captured], step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("ffn", ["gelu", "swiglu"])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_ffn8_gradients_are_the_formula_at_what_is_kept(ext, ffn, dtype):
    """The experts with 8-bit checkpoints against 64 bits on the rows that are kept.

    Pre-activations and the hidden gradient are taken from the GEMMs themselves: a
    different rounding there would move a code by a whole unit.
    """
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(11)
    counts = [0, 37, 1, 90, 0, 72]
    E, A, d, f = len(counts), sum(counts), 96, 160
    off = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32).cuda()
    X = torch.randn(A, d, generator=g).to(dt)
    up = [(torch.randn(E, d, f, generator=g) * d**-0.5).to(dt)
          for _ in range(2 if ffn == "swiglu" else 1)]
    down = (torch.randn(E, f, d, generator=g) * f**-0.5).to(dt)
    dy = torch.randn(A, d, generator=g).to(dt)
    leaves = [t.cuda().requires_grad_() for t in (X, *up, down)]
    fn = moe_ops.swiglu_ffn8_fn if ffn == "swiglu" else moe_ops.grouped_gelu_ffn8_fn
    y = fn(*leaves, off)
    got = [y, *torch.autograd.grad(y, leaves, dy.cuda())]

    seg = np.repeat(np.arange(E), counts)
    X64, up64, down64, dy64 = X.double(), [w.double() for w in up], down.double(), dy.double()

    def rows(a, w):
        return torch.stack([a[i] @ w[seg[i]] for i in range(A)])

    def outer(a, b):
        out = torch.zeros(E, a.shape[1], b.shape[1], dtype=torch.float64)
        for i in range(A):
            out[seg[i]] += torch.outer(a[i], b[i])
        return out

    rnd = lambda t: t.to(dt).double()  # noqa: E731
    if ffn == "swiglu":
        pre = ext.grouped_gemm_swiglu(leaves[0].detach(), off, *(w.detach() for w in leaves[1:3]))[1:]
    else:
        pre = [ext.grouped_gemm_kernel(leaves[0].detach(), off, leaves[1].detach())]
    pre = [p.cpu().double() for p in pre]
    dact = ext.bwd_grouped_gemm_dX_kernel(leaves[-1].detach(), off, dy.cuda()).cpu().double()
    for p, w in zip([*pre, dact], [*up64, down64.transpose(1, 2)]):
        src = dy64 if p is dact else X64
        assert float((p - rows(src, w)).norm() / p.norm()) <= torch.finfo(dt).eps / 2 + 2.0**-18
    act = (lambda a, b: torch.nn.functional.silu(a) * b) if ffn == "swiglu" else _gelu64
    kept = [held64(p).requires_grad_() for p in pre]
    hid = act(*kept)
    dpre = [rnd(t) for t in torch.autograd.grad(hid, kept, dact)]
    Xk = held64(X64)
    dX = sum(rows(t, w.transpose(1, 2)) for t, w in zip(dpre, up64))
    want = [rows(rnd(act(*pre)), down64), dX, *[outer(Xk, t) for t in dpre],
            outer(rnd(hid.detach()), dy64)]
    for name, a, b in zip(("y", "dX", "dW1", "dW2", "dW3"), got, want):
        a = a.detach().cpu().double()
        # The rounding of the hidden rows or of their gradients and the output's own, each
        # at most half a step of the norm; float32 products of up to 160 terms.
        rel = float((a - b).norm() / b.norm())
        assert rel <= torch.finfo(dt).eps + 160 * 2.0**-24, (name, rel)


def test_ffn8_keeps_a_third_of_the_activations(ext):
    """What the backward holds: the point of the checkpoint."""
    A, d, f, E = 4096, 256, 1024, 4
    off = torch.arange(0, A + 1, A // E, dtype=torch.int32).cuda()
    dt = torch.bfloat16
    X = torch.randn(A, d, device="cuda", dtype=dt, requires_grad=True)
    W = [torch.randn(E, d, f, device="cuda", dtype=dt, requires_grad=True) for _ in range(2)]
    out = torch.randn(E, f, d, device="cuda", dtype=dt, requires_grad=True)

    def held(fn):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = fn(X, *W, out, off)
        return torch.cuda.memory_allocated() - before - y.numel() * 2

    # gate, value and X at 33 / 32 bytes a value against 2, and no hidden
    assert held(moe_ops.swiglu_ffn8_fn) <= A * (2 * f + d) * 33 / 32 + 16 * 512
    assert held(moe_ops.swiglu_ffn_fn) >= A * 3 * f * 2


def test_ffn8_frozen_parts(ext):
    """Only the gradients asked for, with the values of the full backward."""
    A, d, f, E = 64, 64, 96, 2
    off = torch.tensor([0, 40, 64], dtype=torch.int32).cuda()
    X = torch.randn(A, d, device="cuda")
    gw, vw = (torch.randn(E, d, f, device="cuda") * 0.1 for _ in range(2))
    ow = torch.randn(E, f, d, device="cuda") * 0.1
    dy = torch.randn(A, d, device="cuda")

    def grads(fn, tensors, on):
        leaves = [t.detach().requires_grad_(o) for t, o in zip(tensors, on)]
        y = fn(*leaves, off)
        return torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy)

    for fn, tensors in ((moe_ops.swiglu_ffn8_fn, (X, gw, vw, ow)),
                        (moe_ops.grouped_gelu_ffn8_fn, (X, gw, ow))):
        n = len(tensors)
        full = grads(fn, tensors, [True] * n)
        for keep in range(1, 2**n - 1):
            on = [bool(keep >> i & 1) for i in range(n)]
            got = grads(fn, tensors, on)
            for a, b in zip(got, [g for g, o in zip(full, on) if o]):
                torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-5)

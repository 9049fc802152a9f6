"""8-bit products at the ends of the documented sizes, and every call of theirs captured."""

import pytest
import torch

from nanotitan_amd import capi, moe_ops
from nanotitan_amd.moe_ops import (
    Int8Weight,
    int8_gelu_ffn_fn,
    int8_grouped_gemm_fn,
    int8_rows,
    int8_rows_decode,
    int8_swiglu_ffn_fn,
    int8_weight,
    int8_weight_decode,
)
from tests import int8_oracle as O
from tests.test_gpu_int8_layer import _case, _check_few

pytestmark = pytest.mark.gpu

U = 2.0**-24


def _rand(*shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


@pytest.mark.parametrize("most", [9, 70])  # streamed weights, tiles
def test_as_many_experts_as_there_may_be(most):
    E, K, N, t = 1024, 70, 66, torch.float16
    g = torch.Generator().manual_seed(most)
    counts = torch.randint(0, most, (E,), generator=g)
    counts[5::7] = 0
    off = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    A, gpu_off = int(off[-1]), off.int().cuda()
    assert (A > 24 * E) == (most == 70)
    W = _rand(E, K, N, seed=1, std=K**-0.5)
    w, x, dout = int8_weight(W), _rand(A, K, dtype=t, seed=2), _rand(A, N, dtype=t, seed=3)
    x.requires_grad_()
    out = int8_grouped_gemm_fn(x, w, gpu_off)
    dx, = torch.autograd.grad(out, x, dout)
    qw, sw = O.held(W.cpu(), 1)
    qx, sx = O.held(x.detach().cpu(), 1)
    want = O.product(qx, sx, qw, sw, off.tolist())
    half, tiny = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal
    assert bool(((out.cpu().double() - want).abs() <= (3.1 * U + half) * want.abs() + tiny).all())
    owner = torch.repeat_interleave(torch.arange(E), counts)
    held, d = (qw.double() * sw.double())[owner], dout.cpu().double().unsqueeze(2)
    want, size = (held @ d).squeeze(2), (held.abs() @ d.abs()).squeeze(2)
    tol = (2.0**-17 + (2 * N + 3) * U) * size + half * want.abs() + tiny
    assert bool(((dx.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_as_many_columns_as_there_may_be(dtype, monkeypatch):
    monkeypatch.setattr(moe_ops, "_int8_direct", lambda d, E, K: True)
    K, N, A = 128, 1 << 22, 130
    g = torch.Generator(device="cuda").manual_seed(1)
    codes = torch.randint(-127, 128, (1, N // 64, K // 64, 4, 4, 16, 16), generator=g,
                          device="cuda", dtype=torch.int8)
    w = Int8Weight(codes, torch.rand(1, N, generator=g, device="cuda") + 0.5, (1, K, N))

    def column(n):  # of integers, in order of k
        c = n % 64
        block = codes[0, n // 64, :, c // 4 % 4, :, 4 * (c // 16) + c % 4]
        return block.reshape(K).cpu().double()

    x = _rand(A, K, dtype=dtype, seed=2).requires_grad_()
    out = int8_grouped_gemm_fn(x, w)
    qx, sx = O.held(x.detach().cpu(), 1)
    half = torch.finfo(dtype).eps / 2
    at = [0, 63, 64, 12345, N // 2 + 1, N - 64, N - 1]
    for n in at:
        want = (qx.double() @ column(n)) * float(w.scale[0, n]) * sx[:, 0].double()
        got = out[:, n].detach().cpu().double()
        assert bool(((got - want).abs() <= (3.1 * U + half) * want.abs()).all())
    # every row has one value of its own, the largest offsets among them
    dout = torch.zeros(A, N, dtype=dtype, device="cuda")
    for r in range(A):
        dout[r, at[r % len(at)]] = 1.0 + r
    del out
    dx, = torch.autograd.grad(int8_grouped_gemm_fn(x, w), x, dout)
    for r in range(A):
        n = at[r % len(at)]
        want = column(n) * float(w.scale[0, n]) * (1.0 + r)
        # of bfloat16 two terms; one product, all others are zeros
        tol = ((2.0**-17 if dtype == torch.bfloat16 else 4 * U) + half + 2 * U) * want.abs()
        assert bool(((dx[r].cpu().double() - want).abs() <= tol).all())


def test_as_long_reductions_as_there_may_be():
    """Gradients of 2^17 columns, forward sums of as many values."""
    K, N, A, t = capi.NT_INT8_MAX_K, 65, 40, torch.bfloat16
    W = _rand(1, K, N, seed=1, dtype=t)
    w, x = int8_weight(W), _rand(A, K, seed=2, dtype=t)
    x.requires_grad_()
    dout = _rand(A, N, seed=3, dtype=t)
    out = int8_grouped_gemm_fn(x, w)
    dx, = torch.autograd.grad(out, x, dout)
    q, s = O.held(W[0].cpu(), 0)
    qx, sx = O.held(x.detach().cpu(), 1)
    half = torch.finfo(t).eps / 2
    want = (qx.double() @ q.double()) * s.double() * sx.double()
    assert bool(((out.cpu().double() - want).abs() <= (3.1 * U + half) * want.abs()).all())
    held, d = q.double() * s.double(), dout.cpu().double()
    want, size = d @ held.t(), d.abs() @ held.abs().t()
    tol = (2.0**-17 + (2 * N + 3) * U) * size + half * want.abs()
    assert bool(((dx.cpu().double() - want).abs() <= tol).all())


def test_as_many_rows_as_there_may_be():
    A, K, N, t = capi.NT_INT8_MAX_ROWS, 8, 9, torch.bfloat16
    w = int8_weight(_rand(1, K, N, seed=1))
    x = torch.zeros(A, K, dtype=t, device="cuda")
    dout = torch.zeros(A, N, dtype=t, device="cuda")
    x[-50:], dout[-50:] = _rand(50, K, dtype=t, seed=2), _rand(50, N, dtype=t, seed=3)
    x.requires_grad_()
    out = int8_grouped_gemm_fn(x, w)
    dx, = torch.autograd.grad(out, x, dout)
    tail = x.detach()[-50:].clone().requires_grad_()
    few = int8_grouped_gemm_fn(tail, w)
    want, = torch.autograd.grad(few, tail, dout[-50:].clone())
    assert torch.equal(out[-50:], few) and torch.equal(dx[-50:], want)
    assert not bool(out[:-50].any()) and not bool(dx[:-50].any())
    for fn in (int8_rows, lambda v: int8_grouped_gemm_fn(v, w)):
        with pytest.raises(RuntimeError):
            fn(torch.zeros(A + 1, K, dtype=t, device="cuda"))


@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("T,d,f,E,k", [(3, 1 << 17, 70, 2, 1), (3, 70, 1 << 17, 2, 2),
                                       (64, 64, 96, 1024, 32), (64, 96, 64, 32, 32)])
def test_few_tokens_at_the_limits(ffn, T, d, f, E, k):
    x, router, w = _case(T, d, f, E, torch.bfloat16, ffn, seed=1)
    _check_few(x, router, None, w, k)


def _steps():
    """name: (step of the static tensors, their refill)."""
    off = torch.tensor([0, 100, 100, 237], dtype=torch.int32, device="cuda")
    E, d, f, A = 3, 200, 264, 237
    W = [_rand(E, d, f, seed=i, std=d**-0.5, dtype=torch.bfloat16) for i in (1, 2)]
    W.append(_rand(E, f, d, seed=3, std=f**-0.5, dtype=torch.bfloat16))
    gate, value, down = [int8_weight(v) for v in W]
    half = _rand(A, d, seed=4, dtype=torch.bfloat16).requires_grad_()
    full = _rand(A, d, seed=5).requires_grad_()
    dy = {n: _rand(A, n, seed=n) for n in (d, f)}
    source = W[0].clone()

    def product(x, exact):
        y = int8_grouped_gemm_fn(x, gate, off, exact_gradient=exact)
        return y.detach(), torch.autograd.grad(y, x, dy[f].to(x.dtype))[0]

    def block(fn, x, *ws, **kw):
        y = fn(x, *ws, off, **kw)
        return y.detach(), torch.autograd.grad(y, x, dy[d].to(x.dtype))[0]

    def weight():
        w = int8_weight(source)
        return w.codes, w.scale, int8_weight_decode(w, torch.bfloat16)

    def rows():
        codes, scales = int8_rows(full)
        return scales, int8_rows_decode(codes, scales, d, torch.float16)

    def refill(*ts):
        def fill(seed):
            with torch.no_grad():
                for t in ts:
                    t.copy_(_rand(*t.shape, seed=seed))
        return fill

    return {"weight": (weight, refill(source)), "rows": (rows, refill(full)),
            "product": (lambda: product(half, True), refill(half)),
            "product rounded": (lambda: product(half, False), refill(half)),
            "product fp32": (lambda: product(full, True), refill(full)),
            "gelu": (lambda: block(int8_gelu_ffn_fn, half, gate, down), refill(half)),
            "gelu rounded": (lambda: block(int8_gelu_ffn_fn, half, gate, down,
                                           exact_gradient=False), refill(half)),
            "gelu fp32": (lambda: block(int8_gelu_ffn_fn, full, gate, down), refill(full)),
            "swiglu fp32": (lambda: block(int8_swiglu_ffn_fn, full, gate, value, down),
                            refill(full))}


@pytest.mark.parametrize("name", ["weight", "rows", "product", "product rounded", "product fp32",
                                  "gelu", "gelu rounded", "gelu fp32", "swiglu fp32"])
def test_captured_and_replayed(name):
    """Each call in a graph, replayed with new inputs between eager calls."""
    step, refill = _steps()[name]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (11, 12, 13, 14):
        refill(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del want

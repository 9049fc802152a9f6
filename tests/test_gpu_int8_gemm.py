"""Products with 8-bit integer weights, and the feed-forward blocks on them, against 64 bits."""

import pytest
import torch

from nanotitan_amd import capi, moe_ops
from nanotitan_amd.moe_ops import (
    Int8Weight,
    int8_gelu_ffn_fn,
    int8_grouped_gemm_fn,
    int8_rows,
    int8_swiglu_ffn_fn,
    int8_weight,
    int8_weight_decode,
)
from tests import int8_oracle as O

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0**-24


def _rand(*shape, dtype=torch.float32, std=1.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()


def _offsets(counts):
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    return off, torch.tensor(off, dtype=torch.int32, device="cuda")


def _weights(E, K, N, seed):
    """(Int8Weight, integers, scales [E,1,N]) of normal weights."""
    W = _rand(E, K, N, std=K**-0.5, seed=seed)
    q, s = O.held(W.cpu(), 1)
    return Int8Weight(O.blocks(q).cuda(), s.view(E, N).cuda(), (E, K, N)), q, s


def _steps(dtype):
    """Half a step of dtype's rounding, relative."""
    return torch.finfo(dtype).eps / 2


# Rows an expert: one, a few, the limits of the row tiles of 16, 32 and 64, of 128 and of 256.
COUNTS = {"one": [1], "eight": [3, 0, 5], "few": [3, 0, 16, 1], "sixteen": [17, 9, 0, 22], "streams": [33, 64, 0, 1],
          "mixed": [200, 0, 3, 50], "tiles": [128, 129, 0, 300], "wide": [256, 1, 700, 513],
          "dense": None}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts", COUNTS)
@pytest.mark.parametrize("K,N", [(128, 64), (300, 65), (1024, 272), (77, 1365)])
def test_product(dtype, counts, K, N):
    t = TYPES[dtype]
    if COUNTS[counts] is None:
        off, gpu_off, E, A = [0, 19], None, 1, 19
    else:
        off, gpu_off = _offsets(COUNTS[counts])
        E, A = len(off) - 1, off[-1]
    x = _rand(A, K, dtype=t, seed=1)
    w, qw, sw = _weights(E, K, N, 2)
    got = int8_grouped_gemm_fn(x, w, gpu_off)
    assert got.dtype == t and got.shape == (A, N)
    qx, sx = O.held(x.cpu(), 1)
    want = O.product(qx, sx, qw, sw, off)
    # the sum to float32 and two products, each half a step, then the output's rounding
    tol = (3.1 * U + _steps(t)) * want.abs() + torch.finfo(t).smallest_normal
    err = (got.cpu().double() - want).abs() - tol
    assert bool((err <= 0).all()), float(err.max())


@pytest.mark.parametrize("rows", [5, 40, 100, 600])
def test_rows_behind_the_last_stay(rows):
    """Rows past offsets[E] are not written, by any of the kernels."""
    E, K, N, A = 3, 200, 130, rows + 37
    off, gpu_off = _offsets([rows // 2, 0, rows - rows // 2])
    x = _rand(A, K, dtype=torch.bfloat16, seed=3)
    codes, scales = int8_rows(x)
    w, _, _ = _weights(E, K, N, 4)
    outs = [torch.full((A, N), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    outs.append(torch.full((A, N), 7.0, device="cuda"))
    s = capi.current_stream()
    args = [capi.NT_BF16, codes.data_ptr(), scales.data_ptr(), gpu_off.data_ptr(),
            w.codes.data_ptr(), w.scale.data_ptr()]
    sizes = [E, A, K, N]
    capi.call("nt_int8_grouped_gemm", *args, *sizes, outs[0].data_ptr(), s)
    capi.call("nt_int8_grouped_gemm_gelu", *args, *sizes, outs[1].data_ptr(), outs[2].data_ptr(), s)
    for o in outs:
        assert bool((o[rows:] == 7.0).all()) and not bool((o[:rows] == 7.0).all())
    outs = [torch.full((A, N), 7.0, dtype=t, device="cuda")
            for t in (torch.bfloat16, torch.float32, torch.float32)]
    capi.call("nt_int8_grouped_gemm_swiglu", *args, w.codes.data_ptr(), w.scale.data_ptr(), *sizes,
              *[o.data_ptr() for o in outs], s)
    for o in outs:
        assert bool((o[rows:] == 7.0).all()) and not bool((o[:rows] == 7.0).all())


def test_no_rows():
    w, _, _ = _weights(2, 64, 96, 0)
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert int8_grouped_gemm_fn(torch.zeros(0, 64, device="cuda"), w, off).shape == (0, 96)
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    out = int8_grouped_gemm_fn(x, w, off)
    out.sum().backward()
    assert x.grad.shape == (0, 64)


def test_malformed_offsets_stay_inside():
    """Offsets that fall, or lie outside [0, A], move no access out of the tensors."""
    w, _, _ = _weights(4, 128, 64, 0)
    for A in (5, 30, 300, 2000):
        x = _rand(A, 128, dtype=torch.bfloat16)
        for off in ([-5, A + 9, 3, 2**31 - 1, 10], [A, 0, A, 0, A], [7, 7, 7, 7, 7]):
            o = torch.tensor(off, dtype=torch.int32, device="cuda")
            assert int8_grouped_gemm_fn(x, w, o).shape == (A, 64)
    torch.cuda.synchronize()


@pytest.mark.parametrize("A", [3, 20, 50, 150, 400])
def test_infinite_and_nan_rows_stay_their_own(A):
    """A row with an infinity or a NaN is NaN; the others are as without it. A NaN channel is a
    NaN column."""
    w, _, _ = _weights(1, 200, 100, 5)
    x = _rand(A, 200, dtype=torch.bfloat16, seed=6)
    want = int8_grouped_gemm_fn(x, w)
    bad = x.clone()
    bad[0, 3], bad[2, 199] = float("inf"), float("nan")
    got = int8_grouped_gemm_fn(bad, w)
    assert bool(got[0].isnan().all()) and bool(got[2].isnan().all())
    keep = [i for i in range(A) if i not in (0, 2)]
    assert torch.equal(got[keep], want[keep])
    scale = w.scale.clone()
    scale[0, 37] = float("nan")
    got = int8_grouped_gemm_fn(x, w._replace(scale=scale))
    assert bool(got[:, 37].isnan().all())
    cols = [i for i in range(100) if i != 37]
    assert torch.equal(got[:, cols], want[:, cols])


def test_the_largest_sums():
    """127 * 127 over the longest reduction is an int32 sum without overflow."""
    K = capi.NT_INT8_MAX_K
    W = torch.ones(1, K, 64, device="cuda")
    w = int8_weight(W)
    for A in (1, 70, 300):
        x = torch.ones(A, K, dtype=torch.float32, device="cuda")
        got = int8_grouped_gemm_fn(x, w)
        one = (torch.tensor(1.0) / 127.0).double()
        want = 127.0 * 127.0 * K * one * one
        assert bool(((got.cpu().double() - want).abs() <= 3.1 * U * want).all())


@pytest.mark.parametrize("A,K", [(8, 2048), (8, 2049), (9, 1700), (4, 4096), (4, 4097), (1, 16384),
                                 (1, 16385), (7, 2300)])
def test_few_rows_are_rounded_as_many(A, K):
    """Rows that the product brings to integers itself, in LDS, and just past those."""
    w, _, _ = _weights(2, K, 130, 12)
    x = _rand(80, K, dtype=torch.bfloat16, seed=13)
    off = torch.tensor([0, A, A], dtype=torch.int32, device="cuda")
    codes, scales = int8_rows(x)
    want = torch.empty(80, 130, dtype=torch.bfloat16, device="cuda")
    many = torch.tensor([0, 80, 80], dtype=torch.int32, device="cuda")
    capi.call("nt_int8_grouped_gemm", capi.NT_BF16, codes.data_ptr(), scales.data_ptr(),
              many.data_ptr(), w.codes.data_ptr(), w.scale.data_ptr(), 2, 80, K, 130,
              want.data_ptr(), capi.current_stream())
    assert torch.equal(int8_grouped_gemm_fn(x[:A], w, off), want[:A])


def test_a_row_is_the_same_in_any_batch():
    w, _, _ = _weights(1, 500, 300, 7)
    x = _rand(700, 500, dtype=torch.bfloat16, seed=8)
    whole = int8_grouped_gemm_fn(x, w)
    for n in (1, 5, 8, 9, 17, 40, 100, 257):
        assert torch.equal(int8_grouped_gemm_fn(x[:n], w), whole[:n])


def test_past_32_bit_offsets():
    """Outputs past 2^31 values and weights past 2^32 bytes."""
    A, K, N = 2**18 + 3, 128, 8256
    w, _, _ = _weights(1, K, N, 9)
    x = _rand(A, K, dtype=torch.bfloat16, seed=10)
    out = int8_grouped_gemm_fn(x, w)
    assert torch.equal(out[-70:], int8_grouped_gemm_fn(x[-70:], w))
    del out
    E, K, N = 34, 16384, 8192
    codes = torch.zeros(E, N // 64, K // 64, 4, 4, 16, 16, dtype=torch.int8, device="cuda")
    codes[-1].random_(-127, 128)
    scale = torch.rand(E, N, device="cuda")
    for rows in (9, 100, 300):
        off = torch.tensor([0] * E + [rows], dtype=torch.int32, device="cuda")
        x = _rand(rows, K, dtype=torch.bfloat16, seed=11)
        got = int8_grouped_gemm_fn(x, Int8Weight(codes, scale, (E, K, N)), off)
        one = Int8Weight(codes[-1:].contiguous(), scale[-1:].contiguous(), (1, K, N))
        assert torch.equal(got, int8_grouped_gemm_fn(x, one))


# ------------------------------------------------------------- feed-forward


def _act64(ffn, pre):
    if ffn == "swiglu":
        return torch.nn.functional.silu(pre[0]) * pre[1]
    return torch.nn.functional.gelu(pre[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("counts", ["few", "sixteen", "streams", "mixed", "tiles", "wide"])
def test_hidden_values(dtype, ffn, counts):
    """Both projections, the activation and the product, elementwise."""
    t = TYPES[dtype]
    off, gpu_off = _offsets(COUNTS[counts])
    E, A, K, N = len(off) - 1, off[-1], 300, 333
    x = _rand(A, K, dtype=t, seed=1)
    codes, scales = int8_rows(x)
    qx, sx = O.held(x.cpu(), 1)
    ws = [_weights(E, K, N, 2 + i) for i in range(2 if ffn == "swiglu" else 1)]
    pre = [O.product(qx, sx, q, s, off) for _, q, s in ws]
    outs = [torch.empty(A, N, dtype=t, device="cuda")]
    outs += [torch.empty(A, N, device="cuda") for _ in range(2 if ffn == "swiglu" else 1)]
    handles = [p for w, _, _ in ws for p in (w.codes.data_ptr(), w.scale.data_ptr())]
    capi.call(f"nt_int8_grouped_gemm_{ffn}", capi.dtype_code(t), codes.data_ptr(),
              scales.data_ptr(), gpu_off.data_ptr(), *handles, E, A, K, N,
              *[o.data_ptr() for o in outs], capi.current_stream())
    got = [o.cpu().double() for o in outs]
    half, tiny = _steps(t), torch.finfo(t).smallest_normal
    err = 3.1 * U  # of a pre-activation, relative
    if ffn == "swiglu":
        for g, p in zip(got[1:], pre):
            assert bool(((g - p).abs() <= err * p.abs() + tiny).all())
        # silu'(z) z is at most (1 + |z|) |silu(z)|; its exponential and reciprocal add a few
        # steps of 2^-24 (e^-z from a float32 product: |z| 2^-23 more)
        slack = err * (2 + pre[0].abs()) + (8 + 2 * pre[0].abs()) * U
    else:
        z = pre[0].requires_grad_()
        cdf = 0.5 * (1 + torch.erf(z.detach() * 0.5**0.5))
        slope = torch.autograd.grad(torch.nn.functional.gelu(z).sum(), z)[0]
        z = z.detach()
        pre = [z]
        # |gelu''| <= 0.8, the fit of Phi is off by 1.2e-7 of a tail
        tol = 0.8 * err * z.abs() + 2e-6 * (1 + z.abs()) + tiny
        assert bool(((got[1] - slope).abs() <= tol).all())
        # gelu's relative slope z phi / Phi is below 2 + z^2
        slack = err * (2 + z * z) + 4e-7 + (8 + 2 * z * z) * U + 0 * cdf
    want = _act64(ffn, pre)
    tol = (slack + half) * want.abs() + tiny
    over = (got[0] - want).abs() - tol
    assert bool((over <= 0).all()), float(over.max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("counts", ["few", "streams", "tiles", "wide", "dense", "one", "three",
                                    "eight"])
def test_block_is_its_stages(dtype, ffn, counts):
    """The feed-forward block has the bits of its stages, each checked above; up to eight rows
    come to 8 bits within the products."""
    t = TYPES[dtype]
    off, gpu_off = ([0, 77], None) if counts == "dense" else _offsets(
        {"three": [1, 0, 2], "eight": [0, 7, 1]}.get(counts) or COUNTS[counts])
    E, A, d, f = len(off) - 1, off[-1], 200, 341
    x = _rand(A, d, dtype=t, seed=1)
    up = [_weights(E, d, f, 2 + i)[0] for i in range(2 if ffn == "swiglu" else 1)]
    down = _weights(E, f, d, 5)[0]
    block = int8_swiglu_ffn_fn if ffn == "swiglu" else int8_gelu_ffn_fn
    y = block(x, *up, down, gpu_off)
    codes, scales = int8_rows(x)
    hidden = torch.empty(A, f, dtype=t, device="cuda")
    handles = [p for w in up for p in (w.codes.data_ptr(), w.scale.data_ptr())]
    capi.call(f"nt_int8_grouped_gemm_{ffn}", capi.dtype_code(t), codes.data_ptr(),
              scales.data_ptr(), None if gpu_off is None else gpu_off.data_ptr(), *handles, E, A,
              d, f, hidden.data_ptr(), *([None] * (2 if ffn == "swiglu" else 1)),
              capi.current_stream())
    assert torch.equal(y, int8_grouped_gemm_fn(hidden, down, gpu_off))


# ----------------------------------------------------------------- gradients


@pytest.fixture(params=["by_size", "direct"])
def direct(request, monkeypatch):
    """Gradients as the sizes choose them (at these, by weights in the tokens' type), and by the
    kernels that read 8-bit weights."""
    if request.param == "direct":
        monkeypatch.setattr(moe_ops, "_int8_direct", lambda d, E, K: True)


def test_which_gradient():
    """Few rows of many weights read them as they are."""
    dout = torch.empty(2000, 4096, dtype=torch.bfloat16, device="meta")
    assert moe_ops._int8_direct(dout, 4, 2048) and not moe_ops._int8_direct(dout, 3, 4096)
    assert not moe_ops._int8_direct(dout, 4, 2047)
    assert moe_ops._int8_direct(dout.float(), 4, 4096)
    assert not moe_ops._int8_direct(dout.float(), 4, 1024)


def _held_weights(ws):
    return [int8_weight_decode(w, torch.float32).cpu().double() for w in ws]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("counts", ["few", "mixed", "wide", "dense"])
@pytest.mark.parametrize("K,N", [(300, 264), (65, 8), (1030, 72), (130, 77), (256, 640)])
def test_product_gradient(dtype, counts, K, N, direct):
    t = TYPES[dtype]
    off, gpu_off = ([0, 19], None) if counts == "dense" else _offsets(COUNTS[counts])
    E, A = len(off) - 1, off[-1]
    x = _rand(A, K, dtype=t, seed=1).requires_grad_()
    w, _, _ = _weights(E, K, N, 2)
    dout = _rand(A, N, dtype=t, seed=3)
    out = int8_grouped_gemm_fn(x, w, gpu_off)
    assert torch.equal(out, int8_grouped_gemm_fn(x.detach(), w, gpu_off))
    out.backward(dout)
    held = _held_weights([w])[0]
    want, size = torch.zeros(A, K).double(), torch.zeros(A, K).double()
    d = dout.cpu().double()
    for e in range(E):
        a, b = off[e], off[e + 1]
        want[a:b] = d[a:b] @ held[e].t()
        size[a:b] = d[a:b].abs() @ held[e].abs().t()
    # the weights' rounding and the output's, half a step each, and a float32 sum of N terms
    tol = (_steps(t) + N * U) * size + _steps(t) * want.abs()
    assert bool(((x.grad.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("counts", ["few", "mixed", "wide", "dense"])
@pytest.mark.parametrize("d,f", [(128, 264), (72, 333), (77, 256), (300, 520)])
def test_block_gradient(dtype, ffn, counts, d, f):
    """dX against the formula in 64 bits, and that against differences."""
    t = TYPES[dtype]
    off, gpu_off = ([0, 19], None) if counts == "dense" else _offsets(COUNTS[counts])
    E, A = len(off) - 1, off[-1]
    x = _rand(A, d, dtype=t, seed=1).requires_grad_()
    up = [_weights(E, d, f, 2 + i)[0] for i in range(2 if ffn == "swiglu" else 1)]
    down = _weights(E, f, d, 5)[0]
    dy = _rand(A, d, dtype=t, seed=6)
    block = int8_swiglu_ffn_fn if ffn == "swiglu" else int8_gelu_ffn_fn
    y = block(x, *up, down, gpu_off)
    assert torch.equal(y, block(x.detach(), *up, down, gpu_off))
    y.backward(dy)
    hu, hd = [_held_weights([w])[0] for w in up], _held_weights([down])[0]
    q, s = O.held(x.detach().cpu(), 1)
    at = (q.double() * s.double()).requires_grad_()

    def smooth(v):  # what the gradient is of: the block at the values held
        return torch.cat([_act64(ffn, [v[a:b] @ h[e] for h in hu]) @ hd[e]
                          for e, (a, b) in enumerate(zip(off, off[1:]))])

    out = smooth(at)
    want = torch.autograd.grad(out, at, dy.cpu().double())[0]
    with torch.no_grad():
        v = _rand(A, d, seed=7).cpu().double()
        diff = ((smooth(at + 1e-6 * v) - smooth(at - 1e-6 * v)) * dy.cpu().double()).sum() / 2e-6
        assert abs(float(diff) - float((want * v).sum())) <= 1e-6 * float(want.norm() * v.norm())
    # 16-bit types: the down projection's weights and the output, half a step of each at most;
    # the terms between are 2^-17, sums of up to 333 float32 products less than 2^-15. float32:
    # the roundings on the way and the sums, below 64 half steps.
    steps = 2 + 2.0**-14 / _steps(t) if t != torch.float32 else 64
    assert float((x.grad.cpu().double() - want).norm()) <= steps * _steps(t) * float(want.norm())


def _terms(t, A, K):
    terms = 3 if t == torch.float32 else 2
    assert capi.load().nt_int8_terms_bytes(capi.dtype_code(t), A, K) == 2 * terms * A * _pitch(K)
    return torch.full((terms, A, _pitch(K)), 7.0, dtype=torch.bfloat16, device="cuda")


def _pitch(K):
    return (K + 127) // 128 * 128


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K,N", [(200, 136), (77, 43), (300, 64)])
def test_terms_of_the_hidden_gradient(dtype, K, N):
    """To 2^-17 or 2^-25 of the value, zeros to a multiple of 16, nothing behind the last row."""
    t, E, rows, A = TYPES[dtype], 3, 150, 180
    off, gpu_off = [0, 100, 100, 150], _offsets([100, 0, 50])[1]
    w, _, _ = _weights(E, K, N, 4)
    dout = torch.zeros(A, (N + 7) // 8 * 8, dtype=t, device="cuda")
    dout[:, :N] = _rand(A, N, dtype=t, seed=1)
    kept = [_rand(A, K, seed=i) for i in (2, 3)]
    scales = [_rand(E, K, seed=i).abs() + 1e-5 for i in (5, 6)]
    terms = [_terms(t, A, K) for _ in range(3)]
    tail, s = [E, A, K, N], capi.current_stream()
    rows_in = dout
    if t == torch.float32:
        rows_in = _terms(t, A, N)
        dense = dout[:, :N].contiguous()
        capi.call("nt_int8_terms", dense.data_ptr(), gpu_off.data_ptr(), w.scale.data_ptr(), E, A,
                  N, rows_in.data_ptr(), s)
        assert bool((rows_in[:, :, N:(N + 15) // 16 * 16] == 0.0).all())
        want = dense.cpu().double() * w.scale.cpu().double()[[0] * 100 + [2] * 80]
        err = (rows_in[:, :, :N].cpu().double().sum(0) - want).abs() - (2.0**-25 + U) * want.abs()
        assert float(err.max()) <= 2.0**-120
    head = [capi.dtype_code(t), w.codes.data_ptr(), w.scale.data_ptr(), gpu_off.data_ptr(),
            rows_in.data_ptr(), dout.shape[1]]
    capi.call("nt_int8_grouped_gemm_dx_gelu", *head, kept[0].data_ptr(), scales[0].data_ptr(),
              *tail, terms[0].data_ptr(), s)
    capi.call("nt_int8_grouped_gemm_dx_swiglu", *head, *[v.data_ptr() for v in kept + scales],
              *tail, terms[1].data_ptr(), terms[2].data_ptr(), s)
    held = int8_weight_decode(w, torch.float32).cpu().to(t).double()
    d, size = torch.zeros(A, K).double(), torch.zeros(A, K).double()
    g = dout[:, :N].cpu().double()
    for e in range(E):
        a, b = off[e], off[e + 1]
        d[a:b] = g[a:b] @ held[e].t()
        size[a:b] = g[a:b].abs() @ held[e].abs().t()
    z, v = [k.cpu().double() for k in kept]
    sg = torch.sigmoid(z)
    owner = torch.tensor([0] * 100 + [2] * 50 + [0] * 30)
    sc = [c.cpu().double()[owner] for c in scales]
    for got, factor in zip(terms, (z * sc[0], v * sg * (1 + z * (1 - sg)) * sc[0], z * sg * sc[1])):
        assert bool((got[:, rows:] == 7.0).all())
        assert bool((got[:, :rows, K:(K + 15) // 16 * 16] == 0.0).all())
        sums = got[:, :rows, :K].cpu().double().sum(0)
        # the terms, the float32 sum, the operations after it with the hardware's exponential and
        # reciprocal; of SwiGLU's slope 1 + z (1 - sg) also where it cancels
        f = factor[:rows]
        tol = (2.0**-17 + (N + 24) * U if t != torch.float32 else (3 * N + 26) * U) \
            * size[:rows] * f.abs()
        tol += 24 * U * (size * (v * sc[0]).abs() * (1 + z.abs()))[:rows]
        want = d[:rows] * f
        err = (sums - want).abs() - tol
        assert bool((err <= 2.0**-100).all()), float(err.max())


def test_gradient_rows_behind_the_last_stay():
    E, K, N, rows, A = 3, 200, 136, 150, 180
    _, off = _offsets([100, 0, 50])
    w, _, _ = _weights(E, K, N, 4)
    dout = _rand(A, N, dtype=torch.bfloat16, seed=1)
    outs = [torch.full((A, K), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
    terms = _terms(torch.bfloat16, A, N)
    terms[:, :rows] = 0.5
    tail, s = [E, A, K, N], capi.current_stream()
    o, p, c = off.data_ptr(), [t.data_ptr() for t in outs], w.codes.data_ptr()
    capi.call("nt_int8_grouped_gemm_dx", capi.NT_BF16, c, w.scale.data_ptr(), o, dout.data_ptr(),
              N, *tail, p[0], s)
    capi.call("nt_int8_grouped_gemm_dx_terms", capi.NT_BF16, c, None, o, terms.data_ptr(), None,
              *tail, p[1], s)
    capi.call("nt_int8_grouped_gemm_dx_terms", capi.NT_BF16, c, c, o, terms.data_ptr(),
              terms.data_ptr(), *tail, p[2], s)
    for t in outs:
        assert bool((t[rows:] == 7.0).all()) and not bool((t[:rows] == 7.0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
def test_block_of_no_rows_and_of_a_sum(dtype, ffn):
    """A gradient of no rows, and one that is a single value seen as all of them."""
    t, f, d = TYPES[dtype], 96, 70
    up = [_weights(2, d, f, i)[0] for i in range(2 if ffn == "swiglu" else 1)]
    down = _weights(2, f, d, 5)[0]
    block = int8_swiglu_ffn_fn if ffn == "swiglu" else int8_gelu_ffn_fn
    for counts in ([0, 0], [0, 9]):
        _, off = _offsets(counts)
        x = _rand(sum(counts), d, dtype=t, seed=3).requires_grad_()
        y = block(x, *up, down, off)
        got, = torch.autograd.grad(y.sum(), x, retain_graph=True)
        want, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert got.shape == x.shape and torch.equal(got, want)


def test_gradient_of_wider_rows():
    """Columns past the next multiple of 8 are not read."""
    E, A, K, N = 2, 50, 90, 43
    w, _, _ = _weights(E, K, N, 4)
    _, off = _offsets([20, 30])
    dout = _rand(A, N, dtype=torch.bfloat16, seed=1)
    outs = []
    for pitch in (48, 64, 136):
        rows = torch.full((A, pitch), float("nan"), dtype=torch.bfloat16, device="cuda")
        rows[:, :48] = 0.0
        rows[:, :N] = dout
        dx = torch.empty(A, K, dtype=torch.bfloat16, device="cuda")
        capi.call("nt_int8_grouped_gemm_dx", capi.NT_BF16, w.codes.data_ptr(), w.scale.data_ptr(),
                  off.data_ptr(), rows.data_ptr(), pitch, E, A, K, N, dx.data_ptr(),
                  capi.current_stream())
        outs.append(dx)
    assert bool(outs[0].isfinite().all()) and all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradient_of_malformed_offsets_stays_inside(dtype):
    t, A, K, N = TYPES[dtype], 300, 130, 64
    ext = moe_ops.get_hip_extension()
    w, v = _weights(4, K, N, 0)[0], _weights(4, N, K, 1)[0]
    dout, kept = _rand(A, N, dtype=t), _rand(A, K)
    for off in ([-5, A + 9, 3, 2**31 - 1, 10], [A, 0, A, 0, A], [7, 7, 7, 7, 7]):
        o = torch.tensor(off, dtype=torch.int32, device="cuda")
        assert ext.int8_dx(dout, o, w.codes, w.scale, K).shape == (A, K)
        terms = ext.int8_dx_gelu(dout, kept, o, w.codes, w.scale, v.scale, K)
        assert ext.int8_dx_terms(terms, None, o, v.codes, v.scale, None, N, t).shape == (A, N)
    torch.cuda.synchronize()


def test_gradient_of_any_alignment_and_layout(direct):
    w, _, _ = _weights(1, 100, 64, 0)
    x = _rand(33, 100, dtype=torch.bfloat16).requires_grad_()
    dout = _rand(33, 64, dtype=torch.bfloat16, seed=1)
    want, = torch.autograd.grad(int8_grouped_gemm_fn(x, w), x, dout)
    buf = torch.empty(33 * 64 + 3, dtype=torch.bfloat16, device="cuda")
    shifted = buf[3:].view(33, 64).copy_(dout)
    turned = dout.t().contiguous().t()
    for g in (shifted, turned):
        got, = torch.autograd.grad(int8_grouped_gemm_fn(x, w), x, g)
        assert torch.equal(got, want)


def test_gradient_at_the_last_of_many_weights():
    """The last expert's weights, past 2^32 bytes."""
    E, K, N = 34, 16384, 8192
    codes = torch.zeros(E, N // 64, K // 64, 4, 4, 16, 16, dtype=torch.int8, device="cuda")
    codes[-1].random_(-127, 128)
    scale = torch.rand(E, N, device="cuda")
    off = torch.tensor([0] * E + [90], dtype=torch.int32, device="cuda")
    x = _rand(90, K, dtype=torch.bfloat16).requires_grad_()
    dout = _rand(90, N, dtype=torch.bfloat16, seed=1)
    got, = torch.autograd.grad(int8_grouped_gemm_fn(x, Int8Weight(codes, scale, (E, K, N)), off),
                               x, dout)
    one = Int8Weight(codes[-1:].contiguous(), scale[-1:].contiguous(), (1, K, N))
    want, = torch.autograd.grad(int8_grouped_gemm_fn(x, one), x, dout)
    assert torch.equal(got, want)


def test_gradients_are_once_differentiable_and_have_no_tangents(direct):
    w, _, _ = _weights(1, 64, 64, 0)
    x = _rand(5, 64).requires_grad_()
    for fn in (lambda v: int8_grouped_gemm_fn(v, w), lambda v: int8_gelu_ffn_fn(v, w, w),
               lambda v: int8_swiglu_ffn_fn(v, w, w, w)):
        g, = torch.autograd.grad(fn(x).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once differentiable"):
            g.square().sum().backward()
        with torch.autograd.forward_ad.dual_level(), torch.no_grad():
            dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(dual)


# ------------------------------------------------- streams, graphs, devices


def test_on_another_stream_and_two_at_once():
    E, d, f = 4, 256, 512
    off, gpu_off = _offsets([100, 0, 37, 300])
    x = [_rand(437, d, dtype=torch.bfloat16, seed=i) for i in (1, 2)]
    up, val, down = (_weights(E, *s, i)[0] for i, s in enumerate([(d, f), (d, f), (f, d)]))
    want = [int8_swiglu_ffn_fn(v, up, val, down, gpu_off) for v in x]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(int8_swiglu_ffn_fn(x[i], up, val, down, gpu_off))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("rows", [5, 150, 600])
def test_captured_and_replayed(rows):
    E, d, f = 2, 256, 384
    off, gpu_off = _offsets([rows, rows // 2])
    A = off[-1]
    up, val, down = (_weights(E, *s, i)[0] for i, s in enumerate([(d, f), (d, f), (f, d)]))
    x = _rand(A, d, dtype=torch.bfloat16, seed=1)
    dy = _rand(A, d, dtype=torch.bfloat16, seed=2)
    leaf = x.clone().requires_grad_()

    def step():
        y = int8_swiglu_ffn_fn(leaf, up, val, down, gpu_off)
        g, = torch.autograd.grad(y, leaf, dy)
        return y.detach(), g

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (3, 4, 5):
        with torch.no_grad():
            leaf.copy_(_rand(A, d, dtype=torch.bfloat16, seed=seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del want


def test_weights_that_would_need_a_gradient_are_refused():
    w, _, _ = _weights(1, 64, 64, 0)
    x = _rand(5, 64)
    with pytest.raises(RuntimeError, match="no gradient"):
        int8_grouped_gemm_fn(x, w._replace(scale=w.scale.clone().requires_grad_()))


def test_refusals():
    w, _, _ = _weights(2, 64, 96, 0)
    x, off = _rand(5, 64), torch.tensor([0, 2, 5], dtype=torch.int32, device="cuda")
    for bad in (lambda: int8_grouped_gemm_fn(x, w), lambda: int8_grouped_gemm_fn(x.double(), w, off),
                lambda: int8_grouped_gemm_fn(x, w, off[:2]),
                lambda: int8_grouped_gemm_fn(x, w, off.long()),
                lambda: int8_grouped_gemm_fn(x, w, off.cpu()),
                lambda: int8_grouped_gemm_fn(x.cpu(), w, off),
                lambda: int8_grouped_gemm_fn(x, w._replace(scale=w.scale.double()), off),
                lambda: int8_grouped_gemm_fn(x, w._replace(codes=w.codes.float()), off),
                lambda: int8_grouped_gemm_fn(x, w._replace(codes=w.codes[:1]), off)):
        with pytest.raises(RuntimeError):
            bad()

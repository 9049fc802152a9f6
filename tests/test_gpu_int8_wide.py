"""The kernels that 8-bit products take at large sizes, against 64 bits at sampled rows and columns
and, in every bit, against the same rows in small calls, which take other kernels."""

import ctypes

import pytest
import torch

from nanotitan_amd import capi, moe_ops
from nanotitan_amd.moe_ops import (
    int8_gelu_ffn_fn,
    int8_grouped_gemm_fn,
    int8_rows,
    int8_swiglu_ffn_fn,
    int8_weight,
    int8_weight_decode,
    moe_few_tokens,
)
from tests import int8_oracle as O
from tests.test_gpu_int8_rows import _check_rows, _values

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0**-24
CHUNK = 1500  # rows of a small call


def _tile(product, E, A, K, N):
    rows, cols = ctypes.c_int32(), ctypes.c_int32()
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    capi.call("nt_int8_tile", product, E, A, K, N, cus, ctypes.byref(rows), ctypes.byref(cols))
    return rows.value, cols.value


def _rand(*shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)


def _offsets(counts):
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    return off, torch.tensor(off, dtype=torch.int32, device="cuda")


def _sample(off):
    """Rows at the ends of the experts and of tiles of 128 and 256, and their experts."""
    rows, owners = [], []
    for e, (a, b) in enumerate(zip(off, off[1:])):
        at = {r for t in range(0, b - a, 1024) for r in (a + t, a + t + 127, a + t + 128, a + t + 255)}
        at = sorted({r for r in (*at, a, a + 1, b - 1, b - 17) if a <= r < b})
        rows += at
        owners += [e] * len(at)
    return rows, owners


def _columns(N):
    return sorted({n for t in range(0, N, 512) for n in (t, t + 63, t + 64, t + 127, t + 128, t + 255)
                   if n < N} | {N - 1, N - 2, N - 65})


def _small(off):
    """Row ranges of at most CHUNK rows with the offsets of their own."""
    for e, (a, b) in enumerate(zip(off, off[1:])):
        for r in range(a, b, CHUNK):
            n = min(CHUNK, b - r)
            yield r, r + n, torch.tensor([0] * (e + 1) + [n] * (len(off) - 1 - e),
                                         dtype=torch.int32, device="cuda")


def _product64(x, Ws, rows, owners, columns):
    """Pre-activations in float64 of sampled rows and columns, one for each of the weights."""
    qx, sx = O.held(x[rows].cpu(), 1)
    out = []
    for W in Ws:
        q, s = O.held(W[:, :, columns].float().cpu(), 1)  # a channel's scale is its column's own
        out.append(torch.stack([(qx[i].double() @ q[e].double()) * s[e, 0].double() * sx[i].double()
                                for i, e in enumerate(owners)]))
    return out


WIDE = {  # product, E's rows, K, N, the tile
    "plain 128x256": ("plain", [4000, 0, 129, 5001, 3000], 333, 1999, (128, 256)),
    "swiglu 128x256": ("swiglu", [4000, 0, 129, 5001, 3000], 333, 1999, (128, 256)),
    "gelu 128x256": ("gelu", [4000, 0, 129, 5001, 3000], 333, 1999, (128, 256)),
    "plain 256x256": ("plain", [5000, 1, 0, 6999, 4100], 8200, 4001, (256, 256)),
    "swiglu 256x256": ("swiglu", [5000, 1, 0, 6999, 4100], 4100, 2001, (256, 256)),
    "gelu 256x256": ("gelu", [5000, 1, 0, 6999, 4100], 8200, 4001, (256, 256)),
}
PRODUCTS = {"plain": capi.NT_INT8_PLAIN, "swiglu": capi.NT_INT8_SWIGLU, "gelu": capi.NT_INT8_GELU}


def _forward(product, x, ws, off, N):
    """The product's outputs through the C ABI: out, or hidden and what a backward needs."""
    t, A, E = x.dtype, x.shape[0], off.numel() - 1
    codes, scales = int8_rows(x)
    outs = [torch.empty(A, N, dtype=t, device="cuda")]
    outs += [torch.empty(A, N, device="cuda")
             for _ in range({"plain": 0, "swiglu": 2, "gelu": 1}[product])]
    handles = [p for w in ws for p in (w.codes.data_ptr(), w.scale.data_ptr())]
    name = "nt_int8_grouped_gemm" + ("" if product == "plain" else f"_{product}")
    capi.call(name, capi.dtype_code(t), codes.data_ptr(), scales.data_ptr(), off.data_ptr(),
              *handles, E, A, x.shape[1], N, *[o.data_ptr() for o in outs], capi.current_stream())
    return outs


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", WIDE)
def test_products(dtype, case):
    """More tiles than workgroups, more k-steps than stages, uneven experts and odd widths."""
    t = TYPES[dtype]
    product, counts, K, N, tile = WIDE[case]
    off, gpu_off = _offsets(counts)
    E, A = len(counts), off[-1]
    assert _tile(PRODUCTS[product], E, A, K, N) == tile
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    wide = tile[1] // (2 if product == "swiglu" else 1)
    assert sum(-(-c // tile[0]) for c in counts) * -(-N // wide) > 2 * cus
    x = _rand(A, K, dtype=t, seed=1)
    Ws = [_rand(E, K, N, dtype=torch.bfloat16, seed=2 + i, std=K**-0.5)
          for i in range(2 if product == "swiglu" else 1)]
    ws = [int8_weight(W) for W in Ws]
    outs = _forward(product, x, ws, gpu_off, N)
    rows, owners = _sample(off)
    cols = _columns(N)
    pre = _product64(x, Ws, rows, owners, cols)
    got = [o[rows][:, cols].cpu().double() for o in outs]
    half, tiny, err = torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal, 3.1 * U
    z = pre[0]
    # as for the small kernels: the sum to float32 and two products; the activation's slope and
    # its own float32 steps; one rounding
    if product == "plain":
        want, slack = z, torch.full_like(z, err)
    elif product == "swiglu":
        for g, p in zip(got[1:], pre):
            assert bool(((g - p).abs() <= err * p.abs() + tiny).all())
        want = torch.nn.functional.silu(z) * pre[1]
        slack = err * (2 + z.abs()) + (8 + 2 * z.abs()) * U
    else:
        leaf = z.clone().requires_grad_()
        slope, = torch.autograd.grad(torch.nn.functional.gelu(leaf).sum(), leaf)
        tol = 0.8 * err * z.abs() + 2e-6 * (1 + z.abs()) + tiny
        assert bool(((got[1] - slope).abs() <= tol).all())
        want = torch.nn.functional.gelu(z)
        slack = err * (2 + z * z) + 4e-7 + (8 + 2 * z * z) * U
    over = (got[0] - want).abs() - ((slack + half) * want.abs() + tiny)
    assert bool((over <= 0).all()), float(over.max())
    assert _tile(PRODUCTS[product], E, CHUNK, K, N) != tile
    for a, b, part in _small(off):
        for whole, small in zip(outs, _forward(product, x[a:b], ws, part, N)):
            assert torch.equal(whole[a:b], small)


COUNTS, D, F = [4000, 0, 129, 5001, 3000], 1290, 1501


def _is_wide(E, K):
    """Tiles of 256 columns, and more of them than workgroups (two a CU)."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    tiles = sum(-(-c // 128) for c in COUNTS) * -(-K // 256)
    return (_tile(capi.NT_INT8_GRADIENT, E, sum(COUNTS), K, 1) == (128, 256)
            and _tile(capi.NT_INT8_GRADIENT, E, CHUNK, K, 1) == (128, 128) and tiles > 2 * cus)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("exact", [True, False])
def test_product_gradients(dtype, exact, monkeypatch):
    monkeypatch.setattr(moe_ops, "_int8_direct", lambda d, E, K: True)
    t = TYPES[dtype]
    off, gpu_off = _offsets(COUNTS)
    E, A, N = len(COUNTS), off[-1], 333
    assert _is_wide(E, F)
    w = int8_weight(_rand(E, F, N, seed=1, std=F**-0.5))
    x = _rand(A, F, dtype=t, seed=2).requires_grad_()
    dout = _rand(A, N, dtype=t, seed=3)

    def gradient(v, d, o):
        return torch.autograd.grad(int8_grouped_gemm_fn(v, w, o, exact_gradient=exact), v, d)[0]

    got = gradient(x, dout, gpu_off)
    rows, owners = _sample(off)
    held, d = int8_weight_decode(w, torch.float32).cpu().double(), dout.cpu().double()[rows]
    want = torch.stack([held[e] @ v for e, v in zip(owners, d)])
    size = torch.stack([held[e].abs() @ v.abs() for e, v in zip(owners, d)])
    half = torch.finfo(t).eps / 2
    if t == torch.float32:  # 2^-25 of three terms, sums of 3 N products
        tol = (3 * N + 6) * U * size
    elif exact:  # 2^-17 of two, sums of 2 N, the output's rounding
        tol = (2.0**-17 + (2 * N + 3) * U) * size + half * want.abs()
    else:  # the weights' rounding and the output's
        tol = (half + N * U) * size + half * want.abs()
    assert bool(((got[rows].cpu().double() - want).abs() <= tol).all())
    for a, b, part in _small(off):
        assert torch.equal(gradient(x.detach()[a:b].requires_grad_(), dout[a:b], part), got[a:b])


@pytest.mark.parametrize("dtype,exact", [("bf16", True), ("bf16", False), ("fp16", True),
                                         ("fp16", False), ("fp32", True)])
@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
def test_block_gradients(dtype, ffn, exact):
    """Both of a backward's products on wide tiles, each workgroup with more than one."""
    t = TYPES[dtype]
    off, gpu_off = _offsets(COUNTS)
    E, A = len(COUNTS), off[-1]
    assert _is_wide(E, F) and _is_wide(E, D)
    up = [int8_weight(_rand(E, D, F, seed=1 + i, std=D**-0.5))
          for i in range(2 if ffn == "swiglu" else 1)]
    down = int8_weight(_rand(E, F, D, seed=4, std=F**-0.5))
    x = _rand(A, D, dtype=t, seed=5).requires_grad_()
    dy = _rand(A, D, dtype=t, seed=6)
    block = int8_swiglu_ffn_fn if ffn == "swiglu" else int8_gelu_ffn_fn

    def gradient(v, d, o):
        return torch.autograd.grad(block(v, *up, down, o, exact_gradient=exact), v, d)[0]

    got = gradient(x, dy, gpu_off)
    rows, owners = _sample(off)
    q, s = O.held(x.detach()[rows].cpu(), 1)
    at = (q.double() * s.double()).requires_grad_()
    hu = [int8_weight_decode(w, torch.float32).cpu().double() for w in up]
    hd = int8_weight_decode(down, torch.float32).cpu().double()
    out = []
    for i, e in enumerate(owners):
        z = [at[i] @ h[e] for h in hu]
        hidden = (torch.nn.functional.silu(z[0]) * z[1] if ffn == "swiglu"
                  else torch.nn.functional.gelu(z[0]))
        out.append(hidden @ hd[e])
    want, = torch.autograd.grad(torch.stack(out), at, dy.cpu().double()[rows])
    # the output's half step (and the down projection's weights'); the terms, 2^-17 of each of
    # three, and float32 sums of at most 3,002 products, below 2^-13 together. float32: below 64.
    half = torch.finfo(t).eps / 2
    steps = (1 if exact else 2) + 2.0**-13 / half if t != torch.float32 else 64
    err = (got[rows].cpu().double() - want).norm(dim=1)
    assert bool((err <= steps * half * want.norm(dim=1)).all())
    for a, b, part in _small(off):
        assert torch.equal(gradient(x.detach()[a:b].requires_grad_(), dy[a:b], part), got[a:b])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,f", [(517, 1), (530, 260), (519, 1024), (517, 2049), (514, 4096),
                                    (530, 4097), (521, 8192), (520, 8193), (515, 14336),
                                    (513, 16385), (513, 40001)])
def test_many_rows(dtype, rows, f):
    """Each of the kernels for more than 512 rows, with a part-filled block of 16 at the end and
    rows whose largest value is anywhere: of zeros, with an infinity or a NaN."""
    x = _values(rows, f, dtype=TYPES[dtype], seed=f, shift=1)
    x[5, -1], x[6, f // 2], x[8] = float("inf"), float("nan"), 0.0
    x[rows - 1, f - 1] = 100.0
    x[rows - 2, f // 3] = -100.0
    _check_rows(x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("E,k", [(4, 2), (64, 8)])
def test_a_token_is_the_same_in_any_batch(dtype, ffn, E, k):
    """The layer for few tokens: where the products bring the rows to 8 bits (up to 8 tokens), the
    last expert sums the tokens (up to 16 experts), and neither."""
    d, f = 1000, 1365
    x, router = _rand(64, d, dtype=TYPES[dtype], seed=1), _rand(E, d, seed=2, std=d**-0.5)
    w = [int8_weight(_rand(E, d, f, seed=3 + i, std=d**-0.5))
         for i in range(2 if ffn == "swiglu" else 1)]
    w.append(int8_weight(_rand(E, f, d, seed=5, std=f**-0.5)))
    with torch.no_grad():
        want = moe_few_tokens(x, w, k, router_weight=router)
        for n in (1, 2, 5, 8, 9, 30):
            for a, b in zip(moe_few_tokens(x[:n], w, k, router_weight=router), want):
                assert torch.equal(a, b[:n])

"""The MoE layer for few tokens (moe_few_tokens, MoE.decode) against 64 bits."""

from types import SimpleNamespace

import pytest
import torch

from nanotitan_amd.moe_ops import moe_few_tokens, route_fn

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0**-24


def _inputs(T, d, f, E, dtype, ffn, seed, shift=0):
    g = torch.Generator().manual_seed(seed)

    def t(*shape, std=1.0, dt=dtype):
        n = 1
        for s in shape:
            n *= s
        # `shift` elements into a buffer: any alignment that a view can have
        buf = (torch.randn(n + shift, generator=g) * std).to(dt).cuda()
        return buf[shift:].view(*shape)

    x = t(T, d)
    router = t(E, d, std=d**-0.5, dt=torch.float32)
    up = [t(E, d, f, std=d**-0.5) for _ in range(2 if ffn == "swiglu" else 1)]
    return x, router, (*up, t(E, f, d, std=f**-0.5))


def _oracle(x, logits, weights, k):
    """(out, its size as a sum of magnitudes, gates, ids) in float64."""
    ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :k]
    gates = logits.gather(1, ids).softmax(-1)
    out, mag = torch.zeros_like(x), torch.zeros_like(x)
    for t in range(x.shape[0]):
        for j in range(k):
            w = [m[ids[t, j]].double() for m in weights]
            a = x[t] @ w[0]
            size = x[t].abs() @ w[0].abs()
            if len(w) == 3:
                b = x[t] @ w[1]
                h = torch.nn.functional.silu(a) * b
                # d silu <= 1.1, |silu| <= |a|
                hmag = h.abs() + 1.1 * size * b.abs() + a.abs() * (x[t].abs() @ w[1].abs())
            else:
                h = torch.nn.functional.gelu(a)
                hmag = h.abs() + 1.2 * size
            out[t] += gates[t, j] * (h @ w[-1])
            mag[t] += gates[t, j] * (hmag @ w[-1].abs())
    return out, mag, gates, ids


def _check(x, router, logits, weights, k):
    with torch.no_grad():
        out, gates, ids = moe_few_tokens(x, weights, k, router_weight=router, logits=logits)
    torch.cuda.synchronize()
    assert out.shape == x.shape and out.dtype == x.dtype
    x64 = x.cpu().double()
    l64 = x64 @ router.cpu().double().t() if router is not None else logits.cpu().double()
    want, mag, g64, i64 = _oracle(x64, l64, [w.cpu() for w in weights], k)
    assert torch.equal(ids.cpu().long(), i64)
    # logits: sums of d products, at most d / 64 + 8 of them in a row
    size = x64.abs() @ router.cpu().double().abs().t() if router is not None else l64.abs()
    slack = (x.shape[1] // 64 + 16) * U * float(size.max() if size.numel() else 0) * 2 + 16 * U
    assert float(((gates.cpu().double() - g64) / g64).abs().max()) <= 2 * slack
    got = out.cpu().double()
    eps = torch.finfo(x.dtype).eps
    if x.dtype == torch.float32:
        # every sum's terms, with up to K / 256 + 16 additions in a row, and the gates' slack
        ulps = max(x.shape[1], weights[-1].shape[1]) / 256 + 64
        tol = ulps * U * mag + 2 * slack * want.abs() + eps / 2 * want.abs()
        assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() - tol).max())
    else:
        # at most half a step for the output's rounding and, with weights that do not know
        # the hidden values' roundings, as much for those
        assert float((got - want).norm()) <= (eps + 2 * slack) * float(want.norm()) + 2.0**-24 * float(
            mag.norm())
        tol = eps / 2 * want.abs() + eps / 2 * mag
        assert bool(((got - want).abs() <= tol).all())
    return out, gates, ids


SHAPES = [  # T, d, f, E, k
    (1, 128, 256, 8, 2), (1, 1, 1, 1, 1), (2, 3, 5, 4, 4), (3, 63, 65, 5, 2), (5, 300, 800, 8, 2),
    (16, 128, 341, 16, 4), (17, 192, 130, 2, 1), (31, 96, 64, 64, 8), (33, 72, 200, 3, 2),
    (64, 256, 96, 128, 8), (64, 40, 36, 1, 1), (49, 100, 257, 4, 2), (7, 33, 31, 1024, 32),
    (64, 64, 64, 32, 32), (4, 512, 2048, 16, 2),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("T,d,f,E,k", SHAPES)
def test_shapes(ext, dtype, ffn, T, d, f, E, k):
    x, router, weights = _inputs(T, d, f, E, TYPES[dtype], ffn, T * d + E)
    _check(x, router, None, weights, k)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T", [16, 17, 40, 64])
def test_all_tokens_on_one_expert(ext, dtype, T):
    """Skewed routing: one expert takes every token, the others one or none."""
    x, _, weights = _inputs(T, 128, 192, 16, TYPES[dtype], "swiglu", T)
    logits = torch.randn(T, 16, generator=torch.Generator().manual_seed(1))
    logits[:, 11] += 50.0
    _check(x, None, logits.cuda(), weights, 2)


@pytest.mark.parametrize("dtype,ffn", [("bf16", "swiglu"), ("fp32", "gelu")])
@pytest.mark.parametrize("sizes", [(16, 1), (17, 16), (32, 17), (33, 32, 1), (48, 33), (49, 48, 2),
                                   (64, 49), (64, 64), (64, 64, 64)])
@pytest.mark.parametrize("E", [5, 64])
def test_an_expert_in_several_loads(ext, dtype, ffn, sizes, E):
    """Given numbers of tokens on the last experts: at and past every multiple of 16 rows,
    with few experts (32 rows a load, or 64) and many (16)."""
    T, k = max(sizes), len(sizes)
    x, _, weights = _inputs(T, 72, 80, E, TYPES[dtype], ffn, sum(sizes))
    g = torch.Generator().manual_seed(2)
    logits = torch.randn(T, E, generator=g)
    for i, n in enumerate(sizes):
        # the last n tokens and, for the others, no token of this expert
        logits[:, E - 1 - i] = torch.where(torch.arange(T) >= T - n, 20.0 + i, -20.0)
    _, _, ids = _check(x, None, logits.cuda(), weights, k)
    for i, n in enumerate(sizes):
        assert int((ids == E - 1 - i).sum()) == n


# T, d, f, E, k, skew: by the number of column tiles, 8, 4, 2 and 1 waves take one; long
# reductions take 128 columns at a time; an expert past 16 tokens among many with few
# takes its weights more than once.
LAYOUTS = [(64, 72, 1000, 24, 1, False), (64, 72, 1000, 48, 2, True), (40, 72, 1000, 64, 2, True),
           (64, 72, 1000, 128, 2, True), (12, 1000, 72, 128, 4, False), (33, 1000, 72, 128, 2, True),
           (5, 8192, 4096, 4, 2, False), (30, 8192, 4096, 4, 2, False), (64, 8000, 4100, 4, 3, False),
           (20, 4100, 8000, 4, 2, False), (3, 4096, 8192, 4, 4, False), (9, 64, 4096, 32, 2, False)]


@pytest.mark.parametrize("dtype,ffn", [("bf16", "swiglu"), ("fp16", "gelu"), ("fp32", "swiglu")])
@pytest.mark.parametrize("T,d,f,E,k,skew", LAYOUTS)
def test_every_tile_layout(ext, dtype, ffn, T, d, f, E, k, skew):
    dt = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(T + E)

    def t(*shape, std):
        return (torch.empty(shape, device="cuda").normal_(0, std, generator=g)).to(dt)

    x = t(T, d, std=1.0)
    up = [t(E, d, f, std=d**-0.5) for _ in range(2 if ffn == "swiglu" else 1)]
    weights = (*up, t(E, f, d, std=f**-0.5))
    logits = torch.empty(T, E, device="cuda").normal_(generator=g)
    if skew:
        logits[:, E // 3] += 50.0
        logits[: T // 2, E - 1] += 40.0
    with torch.no_grad():
        out, gates, ids = moe_few_tokens(x, weights, k, logits=logits)
    want_gates, want_ids = route_fn(logits, k)
    assert torch.equal(ids, want_ids)
    want = torch.zeros(T, d, device="cuda", dtype=torch.float64)
    for e in torch.unique(ids).tolist():
        tok, j = torch.nonzero(ids == e, as_tuple=True)
        a = x[tok].double()
        z = a @ weights[0][e].double()
        if ffn == "swiglu":
            h = torch.nn.functional.silu(z) * (a @ weights[1][e].double())
        else:
            h = torch.nn.functional.gelu(z)
        w = want_gates[tok, j].double().unsqueeze(1)
        want.index_add_(0, tok, w * (h @ weights[-1][e].double()))
    # the roundings of the output and of the hidden values, half a step of the norm each at
    # most; float32 sums of d terms, then f, in chains of at most K / 32 + 8 additions, whose
    # errors add up like those of independent roundings
    ulps = (max(d, f) / 32 + 8) * U
    eps = torch.finfo(dt).eps if dt != torch.float32 else 0.0
    err = (out.double() - want).norm(dim=1)
    assert bool((err <= (eps + 8 * ulps) * want.norm(dim=1)).all()), float(
        (err / want.norm(dim=1)).max())
    with torch.no_grad():
        assert torch.equal(moe_few_tokens(x, weights, k, logits=logits)[0], out)


@pytest.mark.parametrize("dtype", TYPES)
def test_any_alignment(ext, dtype):
    for shift in (1, 2, 3):
        x, router, weights = _inputs(6, 72, 136, 8, TYPES[dtype], "swiglu", shift, shift)
        a = _check(x, router, None, weights, 2)
        b = _check(x.clone(), router.clone(), None, tuple(w.clone() for w in weights), 2)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_ties_masks_and_nan_logits_route_as_route_fn(ext):
    """Equal logits go to the lower id; -inf, the lowest value and NaN as in the full path."""
    T, E, k = 9, 70, 5
    logits = torch.randn(T, E, generator=torch.Generator().manual_seed(2))
    logits[0] = 0.5
    logits[1] = -0.0
    logits[1, 3] = 0.0
    logits[2, 5:] = float("-inf")
    logits[3] = torch.finfo(torch.float32).min
    logits[4, ::2] = float("nan")
    logits[5] = float("-inf")
    logits[6, 7] = float("inf")
    logits[7] = float("nan")
    logits[8, 60:] = torch.finfo(torch.float32).min
    x, _, weights = _inputs(T, 32, 48, E, torch.float32, "gelu", 4)
    with torch.no_grad():
        out, gates, ids = moe_few_tokens(x, weights, k, logits=logits.cuda())
        want_gates, want_ids = route_fn(logits.cuda(), k)
    assert torch.equal(ids, want_ids)
    torch.testing.assert_close(gates, want_gates, rtol=1e-6, atol=1e-30, equal_nan=True)
    for t in range(T):
        assert bool(out[t].isnan().any()) == bool(gates[t].isnan().any())


def test_infinities_stay_in_their_token(ext):
    x, router, weights = _inputs(6, 64, 64, 4, torch.bfloat16, "swiglu", 5)
    logits = torch.randn(6, 4, generator=torch.Generator().manual_seed(5)).cuda()
    ref = _check(x, None, logits, weights, 2)[0]
    bad = x.clone()
    bad[2, 10] = float("inf")
    bad[4, 3] = float("nan")
    with torch.no_grad():
        out = moe_few_tokens(bad, weights, 2, logits=logits)[0]
    for t in (0, 1, 3, 5):
        assert torch.equal(out[t], ref[t])
    for t in (2, 4):
        assert not bool(out[t].isfinite().all())


def test_an_expert_that_no_token_chose_is_not_read(ext):
    x, _, weights = _inputs(5, 64, 96, 8, torch.bfloat16, "swiglu", 6)
    logits = torch.randn(5, 8, generator=torch.Generator().manual_seed(6))
    logits[:, 6] = -100.0
    ref = _check(x, None, logits.cuda(), weights, 2)[0]
    for w in weights:
        w[6] = float("nan")
    with torch.no_grad():
        assert torch.equal(moe_few_tokens(x, weights, 2, logits=logits.cuda())[0], ref)


def test_no_tokens_and_refusals(ext):
    x, router, weights = _inputs(4, 64, 96, 8, torch.float32, "swiglu", 7)
    with torch.no_grad():
        out, gates, ids = moe_few_tokens(x[:0], weights, 2, router_weight=router)
        assert out.shape == (0, 64) and gates.shape == ids.shape == (0, 2)
        logits = torch.randn(4, 8, device="cuda")
        many = torch.randn(65, 64, device="cuda")
        for bad in (lambda: moe_few_tokens(x, weights, 2),
                    lambda: moe_few_tokens(x, weights, 2, router_weight=router, logits=logits),
                    lambda: moe_few_tokens(many, weights, 2, router_weight=router),
                    lambda: moe_few_tokens(x, weights, 9, router_weight=router),
                    lambda: moe_few_tokens(x, weights, 0, router_weight=router),
                    lambda: moe_few_tokens(x.double(), weights, 2, router_weight=router),
                    lambda: moe_few_tokens(x.bfloat16(), weights, 2, router_weight=router),
                    lambda: moe_few_tokens(x, weights, 2, router_weight=router.bfloat16()),
                    lambda: moe_few_tokens(x, weights, 2, logits=logits[:, :7]),
                    lambda: moe_few_tokens(x, weights, 2, logits=logits.cpu()),
                    lambda: moe_few_tokens(x.t(), weights, 2, logits=logits),
                    lambda: moe_few_tokens(x, (weights[0], weights[1][:, :, :95], weights[2]), 2,
                                           logits=logits),
                    lambda: moe_few_tokens(x, (weights[0], weights[0]), 2, logits=logits)):
            with pytest.raises(RuntimeError):
                bad()
    with pytest.raises(RuntimeError, match="no backward"):
        moe_few_tokens(x, tuple(w.clone().requires_grad_() for w in weights), 2,
                       router_weight=router)


def test_graph_streams_and_repeats(ext):
    """Replays, a side stream, and two calls at once give the bits of a plain call."""
    x, router, weights = _inputs(12, 256, 512, 8, torch.bfloat16, "swiglu", 8)
    x2 = _inputs(12, 256, 512, 8, torch.bfloat16, "swiglu", 9)[0]

    def call(v):
        with torch.no_grad():
            return moe_few_tokens(v, weights, 2, router_weight=router)

    ref, ref2 = [t.clone() for t in call(x)], [t.clone() for t in call(x2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            a = call(x2)
        b = call(x)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, ref2))
        assert all(torch.equal(p, q) for p, q in zip(b, ref))
    static = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call(static)
    for v, want in ((x2, ref2), (x, ref), (x2, ref2)):
        static.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(captured, want))
        call(x)


def _cfg(**over):
    c = dict(num_experts=8, top_k=2, d_model=128, ffn_in=256, dtype=torch.bfloat16,
             moe_backend="hip", moe_router_dtype=torch.float32, router_alpha=0.01)
    c.update(over)
    return SimpleNamespace(**c)


@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("router", [torch.float32, torch.bfloat16])
def test_decode_is_the_layer_forward(ext, ffn, router):
    from nanotitan_amd.layer import MoE

    torch.manual_seed(0)
    with torch.device("cuda"):
        moe = MoE(_cfg(moe_router_dtype=router), ffn=ffn)
    for p in moe.experts.parameters():
        p.data.normal_(0, p.shape[1] ** -0.5)
    x = torch.randn(3, 7, 128, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        want = moe(x)[0].float()
    got = moe.decode(x)  # grad mode on: no gradients either way
    assert got.shape == x.shape and not got.requires_grad
    # forward rounds the hidden rows, each expert's output and the sum; decode the first
    # and the last: three half steps of the norm at most, and two
    eps = torch.finfo(torch.bfloat16).eps
    assert float((got.float() - want).norm()) <= 2.5 * eps * float(want.norm())
    # strided tokens, one token
    assert torch.equal(moe.decode(x.transpose(0, 1)), got.transpose(0, 1))
    one = moe.decode(x[:1, :1])
    assert float((one.float() - got[:1, :1].float()).norm()) <= eps * float(one.float().norm())
    with pytest.raises(RuntimeError, match="at most"):
        moe.decode(torch.zeros(5, 13, 128, device="cuda", dtype=torch.bfloat16))

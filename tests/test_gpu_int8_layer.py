"""The MoE layer on 8-bit integer experts: few tokens, the module's two paths, a block, a graph."""

from types import SimpleNamespace

import pytest
import torch

from nanotitan_amd import capi
from nanotitan_amd.layer import Int8ExpertFFN, MoE, MoEBlock, moe_forward_from_logits
from nanotitan_amd.moe_ops import int8_weight, int8_weight_decode, moe_few_tokens, route_fn
from tests import int8_oracle as O

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0**-24


def _case(T, d, f, E, dtype, ffn, seed=0):
    g = torch.Generator().manual_seed(seed)

    def t(*shape, std=1.0, dt=dtype):
        return (torch.randn(*shape, generator=g) * std).to(dt).cuda()

    x, router = t(T, d), t(E, d, std=d**-0.5, dt=torch.float32)
    up = [int8_weight(t(E, d, f, std=d**-0.5)) for _ in range(2 if ffn == "swiglu" else 1)]
    return x, router, (*up, int8_weight(t(E, f, d, std=f**-0.5)))


def _oracle(x, logits, weights, k):
    """(out, gates, ids) in float64, the hidden values held in x's dtype."""
    def held(v):
        q, s = O.held(v, 1)
        return q.double() * s.double()

    w = [int8_weight_decode(m, torch.float32).cpu().double() for m in weights]
    x64 = x.cpu().double()
    ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :k]
    gates = logits.gather(1, ids).softmax(-1)
    out = torch.zeros_like(x64)
    for t in range(x.shape[0]):
        for j in range(k):
            m = [v[ids[t, j]] for v in w]
            row = held(x64[t:t + 1])
            a = row @ m[0]
            h = (torch.nn.functional.silu(a) * (row @ m[1]) if len(m) == 3
                 else torch.nn.functional.gelu(a))
            out[t] += gates[t, j] * (held(h.to(x.dtype).double()) @ m[-1])[0]
    return out, gates, ids


def _check_few(x, router, logits, weights, k):
    with torch.no_grad():
        out, gates, ids = moe_few_tokens(x, weights, k, router_weight=router, logits=logits)
    torch.cuda.synchronize()
    assert out.shape == x.shape and out.dtype == x.dtype
    x64 = x.cpu().double()
    l64 = x64 @ router.cpu().double().t() if router is not None else logits.cpu().double()
    want, g64, i64 = _oracle(x, l64, weights, k)
    assert torch.equal(ids.cpu().long(), i64)
    size = x64.abs() @ router.cpu().double().abs().t() if router is not None else l64.abs()
    slack = 2 * ((x.shape[1] // 64 + 16) * U * float(size.max()) * 2 + 16 * U)
    assert float(((gates.cpu().double() - g64) / g64).abs().max()) <= slack
    # The output's rounding, and hidden values on the other side of a border: those are within
    # 2^-20 of it in units of a step, so one in 2^10 of a float32 row's 127 or fewer steps at
    # most, each a step of 1/127 of the row's largest (below 8 of its norm over sqrt(f)): as a
    # norm 8 / 127 / 2^5 in the worst case, 2^-9.
    eps = torch.finfo(x.dtype).eps
    assert float((out.cpu().double() - want).norm()) <= (eps + slack + 2.0**-9) * float(want.norm())
    return out, gates, ids


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("T,d,f,E,k", [(1, 128, 341, 4, 2), (2, 64, 64, 1, 1), (3, 1, 5, 2, 2),
                                       (5, 300, 800, 16, 4), (17, 512, 700, 8, 2),
                                       (33, 256, 96, 128, 8), (64, 130, 257, 4, 4),
                                       (64, 256, 512, 8, 1), (50, 64, 128, 100, 32)])
def test_few_tokens(dtype, ffn, T, d, f, E, k):
    x, router, w = _case(T, d, f, E, TYPES[dtype], ffn, seed=T)
    _check_few(x, router, None, w, k)


@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("T,d,f,E,k", [(8, 512, 256, 64, 8), (8, 2048, 2048, 16, 2),
                                       (8, 256, 2049, 8, 2), (9, 256, 2048, 8, 1),
                                       (4, 4096, 4096, 8, 2), (4, 4096, 4096, 16, 4),
                                       (1, 16384, 200, 17, 17), (1, 128, 16385, 4, 1),
                                       (2, 16, 16, 1024, 32)])
def test_where_the_rows_are_rounded(ffn, T, d, f, E, k):
    """Around the limits of the rows that the products round for themselves, of the experts whose
    sum is made by the last of them, and of the memory that a workgroup then holds."""
    x, router, w = _case(T, d, f, E, torch.bfloat16, ffn, seed=T)
    _check_few(x, router, None, w, k)


def test_logits_of_the_program():
    x, _, w = _case(9, 128, 256, 8, torch.bfloat16, "swiglu")
    logits = torch.randn(9, 8, generator=torch.Generator().manual_seed(1)).cuda()
    logits[3] = 0.0  # ties go to the lower expert
    _check_few(x, None, logits, w, 3)


def test_gates_are_the_routers():
    x, _, w = _case(40, 128, 256, 64, torch.bfloat16, "gelu")
    logits = torch.randn(40, 64, generator=torch.Generator().manual_seed(2)).cuda()
    logits[0, 5], logits[1, :] = float("inf"), -1e30
    logits[2, 7], logits[2, 8] = 0.0, -0.0
    with torch.no_grad():
        _, gates, ids = moe_few_tokens(x, w, 8, logits=logits)
        g, i = route_fn(logits, 8)
    assert torch.equal(ids, i)
    torch.testing.assert_close(gates, g, rtol=1e-6, atol=0.0, equal_nan=True)


def test_every_token_to_one_expert():
    """More rows than one load of the weights takes, and experts without any."""
    for T, E in ((64, 16), (40, 3)):
        x, _, w = _case(T, 128, 192, E, torch.float16, "swiglu")
        logits = torch.zeros(T, E, device="cuda")
        logits[:, E - 1] = 5.0
        _check_few(x, None, logits, w, 1)


def test_no_tokens_and_limits():
    x, router, w = _case(64, 64, 96, 4, torch.bfloat16, "gelu")
    with torch.no_grad():
        out, gates, ids = moe_few_tokens(x[:0], w, 2, router_weight=router)
        assert out.shape == (0, 64) and gates.shape == ids.shape == (0, 2)
        with pytest.raises(RuntimeError, match="at most 64"):
            moe_few_tokens(torch.cat([x, x]), w, 2, router_weight=router)
        with pytest.raises(RuntimeError, match="top_k"):
            moe_few_tokens(x, w, 5, router_weight=router)
        with pytest.raises(RuntimeError, match="exactly one"):
            moe_few_tokens(x, w, 2)


@pytest.mark.parametrize("T", [6, 20])
def test_a_nan_token_stays_its_own(T):
    x, router, w = _case(T, 128, 256, 4, torch.bfloat16, "swiglu")
    logits = (x.float() @ router.t()).contiguous()
    with torch.no_grad():
        want = moe_few_tokens(x, w, 2, logits=logits)[0]
        bad = x.clone()
        bad[4, 9] = float("inf")
        got = moe_few_tokens(bad, w, 2, logits=logits)[0]
    assert bool(got[4].isnan().all())
    keep = [i for i in range(T) if i != 4]
    assert torch.equal(got[keep], want[keep])


def _cfg(dtype, **over):
    c = dict(num_experts=8, top_k=2, d_model=128, ffn_in=256, dtype=dtype, moe_backend="hip",
             moe_router_dtype=torch.float32, router_alpha=0.01)
    c.update(over)
    return SimpleNamespace(**c)


def _moe(dtype, ffn, seed=0, **over):
    torch.manual_seed(seed)
    with torch.device("cuda"):
        m = MoE(_cfg(dtype, **over), ffn=ffn)
    for p in m.experts.parameters():
        p.data.normal_(0, p.shape[1] ** -0.5)
    return m


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
def test_module(dtype, ffn):
    """forward and decode agree, near the layer in full weights, and the router learns."""
    t = TYPES[dtype]
    m = _moe(t, ffn)
    x = torch.randn(4, 10, 128, device="cuda").to(t)
    with torch.no_grad():
        full = m(x)[0].double()
    held = [tuple(p.shape) for p in m.experts.parameters()]
    assert m.quantize_experts() is m and m.quantize_experts() is m
    assert type(m.experts) is Int8ExpertFFN and not list(m.experts.parameters())
    assert [w.shape for w in m.experts.weights()] == held
    with torch.no_grad():
        y = m(x)[0].double()
        few = m.decode(x).double()
    # 8 bits of normal values: steps of at most 5/127 of a standard deviation, 0.29 of one as a
    # deviation, 0.011 for each of four operands (and more of the hidden values, which have longer tails)
    assert float((y - full).norm() / full.norm()) < 0.06
    # the same integers, up to hidden values at a border: the output's roundings and the full
    # path's of the experts' outputs
    assert float((few - y).norm()) <= (2 * torch.finfo(t).eps + 2.0**-9) * float(y.norm())
    xg = x.clone().requires_grad_()
    out, stats = m(xg)
    (out.float().square().sum() + stats.aux_loss).backward()
    assert bool(xg.grad.isfinite().all()) and float(m.router.weight.grad.norm()) > 0


def test_module_moves_and_keeps_its_scales():
    m = _moe(torch.float32, "swiglu").quantize_experts()
    scales = [w.scale.clone() for w in m.experts.weights()]
    state = {k: v.clone() for k, v in m.state_dict().items()}
    m.experts.to(torch.bfloat16)
    m.experts.half()
    assert all(torch.equal(w.scale, s) for w, s in zip(m.experts.weights(), scales))
    other = _moe(torch.float32, "swiglu", seed=1).quantize_experts()
    other.load_state_dict(state)
    x = torch.randn(1, 7, 128, device="cuda")
    with torch.no_grad():
        assert torch.equal(other(x)[0], m(x)[0])
        assert torch.equal(other.decode(x), m.decode(x))


def test_decode_with_hooks():
    """A hook on 8-bit experts runs, by the full path."""
    m = _moe(torch.bfloat16, "gelu").quantize_experts()
    x = torch.randn(1, 6, 128, device="cuda", dtype=torch.bfloat16)
    seen = []
    h = m.experts.register_forward_hook(lambda mod, args, out: seen.append(out.shape))
    m.decode(x)
    assert seen == [(12, 128)]
    h.remove()


def test_block_trains_around_frozen_experts():
    torch.manual_seed(0)
    with torch.device("cuda"):
        block = MoEBlock(_cfg(torch.float32), norm="layer", residual_scale=0.5)
    for p in block.moe.experts.parameters():
        p.data.normal_(0, p.shape[1] ** -0.5)
    block.moe.quantize_experts()
    x = torch.randn(2, 40, 128, device="cuda", requires_grad=True)
    h, _, stats = block(x)
    (h.square().mean() + stats.aux_loss).backward()
    grads = {n: p.grad for n, p in block.named_parameters()}
    assert grads and all(g is not None and bool(g.isfinite().all()) for g in grads.values())
    got, _ = block.decode(x.detach()[:, :5])
    with torch.no_grad():
        want = block(x.detach()[:, :5])[0]
    assert float((got - want).norm()) <= 2.0**-9 * float(want.norm())


def test_gradient_through_the_layer():
    """moe_forward_from_logits on 8-bit experts against the same on the weights they hold."""
    m = _moe(torch.float32, "swiglu")
    e8 = Int8ExpertFFN(m.experts)
    for name, w in zip(e8.names, e8.weights()):
        getattr(m.experts, name).data = int8_weight_decode(w, torch.float32)
    x = torch.randn(60, 128, device="cuda")
    q, s = O.held(x.cpu(), 1)
    x = (q.double() * s.double()).float().cuda()  # values that 8 bits hold
    logits = torch.randn(60, 8, device="cuda")
    dy = torch.randn(60, 128, device="cuda")
    grads = []
    for experts in (e8, m.experts):
        a = [v.clone().requires_grad_() for v in (x, logits)]
        out, _, _ = moe_forward_from_logits(*a, experts, 8, 2)
        grads.append(torch.autograd.grad(out, a, dy))
    # tokens: the same products of the same values; gates: of outputs whose hidden values were
    # rounded to 8 bits, 0.29 steps of 1/127 of a row's largest (at most 12 deviations) as a norm
    assert float((grads[0][0] - grads[1][0]).norm()) <= 1e-4 * float(grads[1][0].norm())
    assert float((grads[0][1] - grads[1][1]).norm()) <= 0.03 * float(grads[1][1].norm())


@pytest.mark.parametrize("T", [1, 6, 40])
def test_captured_and_replayed(T):
    x, router, w = _case(T, 256, 512, 8, torch.bfloat16, "swiglu")
    static = x.clone()
    with torch.no_grad():
        moe_few_tokens(static, w, 2, router_weight=router)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = moe_few_tokens(static, w, 2, router_weight=router)
        for seed in range(4):
            g = torch.Generator().manual_seed(seed)
            static.copy_(torch.randn(T, 256, generator=g).to(torch.bfloat16).cuda())
            graph.replay()
            torch.cuda.synchronize()
            got = [o.clone() for o in out]
            want = moe_few_tokens(static, w, 2, router_weight=router)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_and_a_dirty_workspace():
    x, router, w = _case(30, 128, 256, 8, torch.bfloat16, "swiglu")
    with torch.no_grad():
        want = moe_few_tokens(x, w, 2, router_weight=router)[0]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        got = []
        for _ in range(4):
            for s in streams:
                with torch.cuda.stream(s):
                    got.append(moe_few_tokens(x, w, 2, router_weight=router)[0])
        torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    T, d, f, E, k = 30, 128, 256, 8, 2
    size = capi.load().nt_int8_moe_few_tokens_workspace_bytes(capi.NT_BF16, T, E, k, d, f)
    up, val, down = w
    for fill in (0, 255):
        ws = torch.full((size,), fill, dtype=torch.uint8, device="cuda")
        gates = torch.empty(T, k, device="cuda")
        topk = torch.empty(T, k, dtype=torch.int32, device="cuda")
        out = torch.empty_like(x)
        for _ in range(2):
            capi.call("nt_int8_moe_few_tokens", capi.NT_BF16, x.data_ptr(), router.data_ptr(), None,
                      up.codes.data_ptr(), up.scale.data_ptr(), val.codes.data_ptr(),
                      val.scale.data_ptr(), down.codes.data_ptr(), down.scale.data_ptr(), T, E, k,
                      d, f, gates.data_ptr(), topk.data_ptr(), out.data_ptr(), ws.data_ptr(), size,
                      capi.current_stream())
            assert torch.equal(out, want)

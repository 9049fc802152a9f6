"""The MoE half of a transformer layer: norms, MoE, gate, residual and 8-bit
checkpoints together, in training, under a graph and in decoding."""

from types import SimpleNamespace

import pytest
import torch

from nanotitan_amd.layer import MoEBlock

pytestmark = pytest.mark.gpu


def _cfg(dtype, **over):
    c = dict(num_experts=8, top_k=2, d_model=128, ffn_in=256, dtype=dtype, moe_backend="hip",
             moe_router_dtype=torch.float32, router_alpha=0.01)
    c.update(over)
    return SimpleNamespace(**c)


def _blocks(dtype, n=2, seed=0, **kw):
    torch.manual_seed(seed)
    over = kw.pop("cfg", {})
    with torch.device("cuda"):
        blocks = [MoEBlock(_cfg(dtype, **over), **kw) for _ in range(n)]
    for b in blocks:
        for name, p in b.named_parameters():
            if "experts" in name:
                p.data.normal_(0, p.shape[1] ** -0.5)
            elif "router" not in name:
                p.data.add_(torch.randn_like(p) * 0.2)
    return blocks


def _chain(blocks, x, gate=None):
    normed, aux = None, 0.0
    for b, nxt in zip(blocks, [*blocks[1:], None]):
        x, normed, stats = b(x, normed=normed, gate=gate, following=nxt)
        aux = aux + stats.aux_loss
    return x, aux


def _norm(v, w, b, kind, eps=1e-6):
    if kind == "layer":
        return torch.nn.functional.layer_norm(v, v.shape[-1:], w, b, eps)
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w


def _unfused(blocks, x, gate=None):
    """The same chain with torch norms around the MoE layers."""
    aux = 0.0
    for b in blocks:
        y, stats = b.moe(_norm(x, b.pre_weight, b.pre_bias, b.norm))
        aux = aux + stats.aux_loss
        if b.post_weight is not None:
            y = _norm(y, b.post_weight, b.post_bias, b.norm)
        if gate is not None:
            y = y * gate
        if b.scale is not None:
            y = y * b.scale
        x = x + y
    return x, aux


KINDS = [dict(norm="rms", post_norm=True, residual_scale=0.5),
         dict(norm="layer", post_norm=False),  # the reference's x + ffn(ffn_norm(x))
         dict(norm="layer", post_norm=True, residual_scale=0.1, ffn="gelu")]


@pytest.mark.parametrize("kw", KINDS)
@pytest.mark.parametrize("gated", [False, True])
def test_chain_equals_unfused_float32(ext, kw, gated):
    blocks = _blocks(torch.float32, **kw)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 50, 128, device="cuda", generator=g, requires_grad=True)
    gate = torch.rand(3, 50, 128, device="cuda", generator=g).requires_grad_() if gated else None
    dy = torch.randn(3, 50, 128, device="cuda", generator=g)
    leaves = [x, *([gate] if gated else []), *[p for b in blocks for p in b.parameters()]]

    def grads(f):
        out, aux = f(blocks, x, gate)
        return out, torch.autograd.grad([out, aux], leaves, [dy, torch.ones_like(aux)])

    (a, ga), (b, gb) = grads(_chain), grads(_unfused)
    # float32 both ways: 2 layers of sums of up to 256 terms, roundings of the norm
    tol = 4096 * 2.0**-24
    a, b = a.detach(), b.detach()
    assert float((a - b).norm()) <= tol * float(b.norm())
    for p, q in zip(ga, gb):
        assert float((p - q).norm()) <= tol * float(q.norm()) + 1e-7


@pytest.mark.parametrize("kw", KINDS[:2])
def test_checkpoints_change_the_weight_gradients_by_their_rounding(ext, kw):
    """Outputs are the same bits; the gradients move by what 8 bits round away."""
    dtype = torch.bfloat16
    plain = _blocks(dtype, n=1, **kw)[0]
    kept = _blocks(dtype, n=1, cfg=dict(ffn_checkpoint8=True), **kw)[0]
    kept.load_state_dict(plain.state_dict())
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(4, 100, 128, device="cuda", generator=g).to(dtype)
    dy = torch.randn(4, 100, 128, device="cuda", generator=g).to(dtype)
    res = []
    for b in (plain, kept):
        leaf = x.detach().requires_grad_()
        out, _, stats = b(leaf)
        res.append((out, torch.autograd.grad([out, stats.aux_loss], [leaf, *b.parameters()],
                                             [dy, torch.ones_like(stats.aux_loss)])))
    assert torch.equal(res[0][0], res[1][0])
    for p, q in zip(res[0][1], res[1][1]):
        # A unit is at most 2 / 127.5 of its block's largest value, which is below 3.5
        # deviations in 98.5 % of blocks of 32 normal values: 2^-4.2 of the deviation, and
        # 1 / sqrt(12) of that, 2^-6, as the rounding's norm. A gradient multiplies with two
        # rounded factors at most (the hidden rows or X, and the activation's slope).
        assert float((p.float() - q.float()).norm()) <= 2 * 2.0**-5.8 * float(p.float().norm())


def test_training_step_under_graph_replay(ext):
    blocks = _blocks(torch.bfloat16, cfg=dict(ffn_checkpoint8=True), **KINDS[0])
    params = [p for b in blocks for p in b.parameters()]
    x = torch.zeros(2, 64, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn(2, 64, 128, device="cuda").to(torch.bfloat16)

    def step():
        out, aux = _chain(blocks, x)
        grads = torch.autograd.grad([out, aux], [x, *params], [dy, torch.ones_like(aux)])
        # no eager graph of the leaves may live while one is captured
        return [out.detach(), *grads]

    def fill(seed):
        with torch.no_grad():
            x.copy_(torch.randn(2, 64, 128, generator=torch.Generator().manual_seed(seed)))

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("kw", KINDS)
def test_decode_follows_forward(ext, kw):
    """Token by token through decode, eager and captured: the prompt pass's outputs."""
    dtype = torch.bfloat16
    blocks = _blocks(dtype, **kw)
    x = torch.randn(6, 1, 128, device="cuda").to(dtype)
    with torch.no_grad():
        want = _chain(blocks, x)[0].float()

    def decode(v):
        normed = None
        for b, nxt in zip(blocks, [*blocks[1:], None]):
            v, normed = b.decode(v, normed=normed, following=nxt)
        return v

    got = decode(x)
    # 2.5 steps of the MoE's norm a block (see MoE.decode), two blocks, and the second
    # block's MoE follows a moved input: twice that at most
    eps = torch.finfo(dtype).eps
    assert float((got.float() - want).norm()) <= 10 * eps * float(want.norm())
    static = torch.zeros_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = decode(static)
    for _ in range(3):
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, got)
        decode(x)

"""Derivatives that the norms, the 8-bit activations and the few-token layer do not
have are refused, not dropped. Without a GPU: the refusals come before any kernel."""

from types import SimpleNamespace

import pytest
import torch
from torch.autograd import forward_ad

from nanotitan_amd import moe_ops
from nanotitan_amd.layer import MoE

D, F, E = 8, 16, 2


def _calls():
    """name -> (tensors, f(*tensors)), one entry for each input that could carry a tangent."""
    x, w, s = torch.randn(4, D), torch.ones(D), torch.ones(1)
    up, down = torch.randn(E, D, F), torch.randn(E, F, D)
    router, logits = torch.randn(E, D), torch.randn(4, E)
    few = moe_ops.moe_few_tokens
    return {
        "pre_norm": ((x, w, w), lambda a, b, c: moe_ops.pre_norm_fn(a, b, c, kind="layer")),
        "post_norm": ((x, x, w, w, x, s, w, w), lambda a, y, p, b, g, c, n, m: moe_ops.post_norm_fn(
            a, y, p, b, gate=g, scale=c, next_weight=n, next_bias=m, kind="layer")),
        "gelu8": ((x,), moe_ops.gelu8_fn),
        "swiglu8": ((x, x), moe_ops.swiglu8_fn),
        "few_router": ((x, up, down, router), lambda a, u, v, r: few(a, (u, v), 1, r)),
        "few_logits": ((x, up, up, down, logits),
                       lambda a, u, m, v, z: few(a, (u, m, v), 1, logits=z)),
    }


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", list(_calls()))
def test_forward_mode_is_refused(name, grad):
    tensors, f = _calls()[name]
    for i in range(len(tensors)):
        with forward_ad.dual_level(), torch.set_grad_enabled(grad):
            ins = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t
                   for j, t in enumerate(tensors)]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(*ins)


def test_forward_mode_through_decode_is_refused():
    cfg = SimpleNamespace(num_experts=E, top_k=1, d_model=D, ffn_in=F, moe_backend="hip",
                          dtype=torch.float32, router_alpha=0.01)
    moe = MoE(cfg, ffn="gelu")
    x = torch.randn(1, 3, D)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        moe.decode(forward_ad.make_dual(x, torch.ones_like(x)))


def test_tangents_that_are_switched_off_are_no_reason():
    x = torch.randn(4, D)
    with forward_ad.dual_level(), forward_ad._set_fwd_grad_enabled(False):
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="GPU tensor"):
            moe_ops.gelu8_fn(dual)


class _Square(torch.autograd.Function):
    """x^2 with a backward that, like a kernel's, has no graph of its own."""

    @staticmethod
    def forward(ctx, x, scale):
        ctx.save_for_backward(x.detach(), scale.detach())
        return x * x * scale

    @staticmethod
    @moe_ops._once_differentiable
    def backward(ctx, dy):
        x, scale = ctx.saved_tensors
        return 2 * x * scale * dy, None


def test_a_second_derivative_meets_an_error():
    """On the way to the leaf and to the output's gradient, not only in backward()."""
    x, s = torch.tensor([3.0], requires_grad=True), torch.tensor([1.0])
    (g,) = torch.autograd.grad(_Square.apply(x, s).sum(), x, create_graph=True)
    assert float(g) == 6.0
    penalty = (_Square.apply(x, s) + g * g).sum()
    with pytest.raises(RuntimeError, match="once differentiable"):
        torch.autograd.grad(penalty, x, retain_graph=True)
    with pytest.raises(RuntimeError, match="once differentiable"):
        penalty.backward()
    with pytest.raises(RuntimeError, match="once differentiable"):
        torch.autograd.functional.jvp(lambda v: _Square.apply(v, s), x.detach(), torch.ones(1))
    x.grad = None
    _Square.apply(x, s).sum().backward()  # the first is as it was
    assert float(x.grad) == 6.0

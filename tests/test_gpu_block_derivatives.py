"""What the norms', the 8-bit activations' and the few-token layer's kernels refuse of derivatives."""

import pytest
import torch

from nanotitan_amd import moe_ops

pytestmark = pytest.mark.gpu


NAMES = ["pre_norm", "post_norm", "gelu8", "swiglu8", "gelu_ffn8", "swiglu_ffn8"]


def _calls():
    g = torch.Generator(device="cuda").manual_seed(0)

    def t(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    w, up, down = t(64), t(2, 64, 96) * 0.1, t(2, 96, 64) * 0.1
    off = torch.tensor([0, 3, 8], dtype=torch.int32, device="cuda")
    return {
        "pre_norm": lambda x: moe_ops.pre_norm_fn(x, w),
        "post_norm": lambda x: moe_ops.post_norm_fn(x, x, w, next_weight=w)[1],
        "gelu8": moe_ops.gelu8_fn,
        "swiglu8": lambda x: moe_ops.swiglu8_fn(x, x),
        "gelu_ffn8": lambda x: moe_ops.grouped_gelu_ffn8_fn(x, up, down, off),
        "swiglu_ffn8": lambda x: moe_ops.swiglu_ffn8_fn(x, up, up, down, off),
    }


@pytest.mark.parametrize("name", NAMES)
def test_a_gradient_penalty_is_refused(ext, name):
    """A term of the loss that is made of first gradients, which have no graph."""
    f = _calls()[name]
    x = torch.randn(8, 64, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(f(x).sum(), x, create_graph=True)
    (plain,) = torch.autograd.grad(f(x).sum(), x)
    assert torch.equal(g, plain)
    loss = f(x).square().sum() + g.square().sum()
    with pytest.raises(RuntimeError, match="once differentiable"):
        torch.autograd.grad(loss, x, retain_graph=True)
    with pytest.raises(RuntimeError, match="once differentiable"):
        loss.backward()
    with pytest.raises(RuntimeError, match="once differentiable"):
        torch.autograd.functional.jvp(f, x.detach(), torch.ones_like(x))


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(ext, name):
    x = torch.randn(8, 64, device="cuda")
    with pytest.raises(RuntimeError):
        torch.func.jvp(_calls()[name], (x,), (torch.ones_like(x),))

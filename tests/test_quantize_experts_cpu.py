"""What MoE.quantize_experts refuses to lose, without a GPU."""

from types import SimpleNamespace

import pytest
import torch

from nanotitan_amd.layer import MoE

HOOKS = ["register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook",
         "register_full_backward_pre_hook"]


def _moe(ffn):
    cfg = SimpleNamespace(num_experts=2, top_k=1, d_model=8, ffn_in=16, dtype=torch.float32,
                          moe_backend="hip", router_alpha=0.01)
    return MoE(cfg, ffn=ffn)


@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("register", HOOKS)
def test_hooks_on_the_experts(ffn, register):
    m = _moe(ffn)
    before = m.experts
    handle = getattr(before, register)(lambda *args: None)
    with pytest.raises(RuntimeError, match="remove their hooks"):
        m.quantize_experts()
    assert m.experts is before and m.moe_backend.experts is before
    handle.remove()
    with pytest.raises(RuntimeError, match="must be a GPU tensor"):  # and then it goes on
        m.quantize_experts()
    assert m.experts is before


def test_a_forward_in_place_of_the_experts():
    m = _moe("gelu")
    m.experts.forward = lambda x, off: x
    with pytest.raises(RuntimeError, match="remove their hooks"):
        m.quantize_experts()

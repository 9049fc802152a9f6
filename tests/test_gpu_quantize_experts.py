"""What MoE.quantize_experts keeps of the module."""

import copy
import io
from types import SimpleNamespace

import pytest
import torch

from nanotitan_amd.layer import MoE
from nanotitan_amd.moe_ops import int8_rows, int8_weight
from tests import int8_oracle as O

pytestmark = pytest.mark.gpu


def _moe(**over):
    cfg = SimpleNamespace(**{**dict(num_experts=4, top_k=2, d_model=64, ffn_in=96,
                                    dtype=torch.bfloat16, moe_backend="hip", router_alpha=0.01,
                                    moe_router_dtype=torch.float32), **over})
    torch.manual_seed(0)
    with torch.device("cuda"):
        return MoE(cfg)


@pytest.mark.parametrize("training", [True, False])
def test_the_mode_stays(training):
    m = _moe().train(training).quantize_experts()
    assert all(part.training == training for part in m.modules())


def test_copies_and_saved_modules():
    """A copy, and a module restored from its state, give the same and are their own."""
    m = _moe().quantize_experts()
    x = torch.randn(2, 9, 64, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        want = [m(x)[0], m.decode(x)]
        twin = copy.deepcopy(m)
        assert twin.moe_backend.experts is twin.experts and twin.experts is not m.experts
        file = io.BytesIO()
        torch.save(m.state_dict(), file)
        file.seek(0)
        other = _moe().quantize_experts()
        for name in other.experts.names:
            getattr(other.experts, f"{name}_codes").zero_()
        other.load_state_dict(torch.load(file, weights_only=True))
        for name in m.experts.names:
            getattr(m.experts, f"{name}_codes").zero_()
        for again in (twin, other):
            assert torch.equal(again(x)[0], want[0]) and torch.equal(again.decode(x), want[1])


def test_values_that_require_gradients():
    """Parameters, transposed views of them too, go to 8 bits without a graph."""
    p = torch.nn.Parameter(torch.randn(70, 130, device="cuda"))
    for v in (p, p.t()):
        w, (codes, scales) = int8_weight(v), int8_rows(v)
        assert not (w.scale.requires_grad or scales.requires_grad)
        plain = v.detach().clone()
        assert torch.equal(w.codes, int8_weight(plain).codes)
        rows = v.shape[0]  # (those behind the last, up to 16, hold anything)
        assert torch.equal(O.plain_rows(codes)[:rows], O.plain_rows(int8_rows(plain)[0])[:rows])

"""Forward-mode tangents of values that go to 8 bits are refused, not dropped; no GPU needed."""

import pytest
import torch
from torch.autograd import forward_ad

from nanotitan_amd import moe_ops


@pytest.mark.parametrize("fn,shape", [(moe_ops.int8_rows, (4, 64)), (moe_ops.int8_weight, (8, 16)),
                                      (moe_ops.int8_weight, (2, 8, 16))])
@pytest.mark.parametrize("turned", [False, True])
def test_dual_tensors_are_refused(fn, shape, turned):
    v = torch.randn(shape)
    if turned:
        v = v.transpose(-1, -2).contiguous().transpose(-1, -2)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            fn(forward_ad.make_dual(v, torch.ones_like(v)))
    with pytest.raises(RuntimeError, match="must be a GPU tensor"):  # and without one go on
        fn(v.requires_grad_())

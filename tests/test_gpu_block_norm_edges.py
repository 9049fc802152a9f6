"""Block norms where a value is infinite or missing: what the formula says, at every width."""

import pytest
import torch

from nanotitan_amd.moe_ops import post_norm_fn

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
WIDTHS = [5, 8, 13, 200, 203, 2056, 2059, 9001]  # whole chunks of eight columns, and a last one moved back


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gate", ["none", "token", "full"])
@pytest.mark.parametrize("d", WIDTHS)
def test_without_its_norm_a_branch_has_the_gradient_of_a_product(ext, dtype, gate, d):
    """h = x + s g y: dy = s g dh, whatever y holds."""
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(d)
    x, y, dh = (torch.randn(6, d, generator=g).to(dt) for _ in range(3))
    y[2, d // 2], y[3, 0], y[4, d - 1] = float("inf"), float("-inf"), float("nan")
    gt = {"none": None, "token": torch.rand(6, 1, generator=g).to(dt),
          "full": torch.rand(6, d, generator=g).to(dt)}[gate]
    s = torch.tensor([0.5], dtype=dt)
    leaf = y.cuda().requires_grad_()
    for kind in ("rms", "layer"):
        h = post_norm_fn(x.cuda(), leaf, gate=None if gt is None else gt.cuda(), scale=s.cuda(),
                         kind=kind)
        (dy,) = torch.autograd.grad(h, leaf, dh.cuda())
        want = 0.5 * dh.double() * (1.0 if gt is None else gt.double())
        tol = torch.finfo(dt).eps / 2 * want.abs() + 2 * 2.0**-24 * want.abs() + (
            2.0**-25 if dt == torch.float16 else 0.0)  # half a step, two float32 products
        assert bool(((dy.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [w for w in WIDTHS if w > 8])
def test_an_infinite_gate_touches_its_column(ext, dtype, d):
    """rms: the row's r is 0, so n is 0 but for the infinite column's 0 * inf."""
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(d)
    x, y, w = (torch.randn(4, d, generator=g).to(dt).cuda() for _ in range(3))
    y = y.sign() * (y.abs() + 0.5)  # no zero, whose product with it is a NaN
    gate = torch.ones(4, d, dtype=dt, device="cuda")
    for col in range(max(0, d - 9), d):  # the last chunk, and what it moves back over
        g1 = gate.clone()
        g1[1, col] = float("inf")
        h, n = post_norm_fn(x, y, gate=g1, next_weight=w[0], kind="rms")
        assert bool(h[1, col].isinf()) and int((~h.isfinite()).sum()) == 1
        at = torch.zeros(4, d, dtype=torch.bool, device="cuda")
        at[1, col] = True
        assert torch.equal(n.isnan(), at)
        assert int((n[1] != 0).sum()) == 1  # the NaN
        rest = post_norm_fn(x, y, gate=gate, next_weight=w[0], kind="rms")[1]
        assert torch.equal(n[[0, 2, 3]], rest[[0, 2, 3]])

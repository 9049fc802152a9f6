"""MoE.decode runs what a user hung on the experts, as forward does."""

from types import SimpleNamespace

import pytest
import torch

from nanotitan_amd.layer import MoE

pytestmark = pytest.mark.gpu


def _moe(ffn):
    cfg = SimpleNamespace(num_experts=8, top_k=2, d_model=128, ffn_in=256, dtype=torch.bfloat16,
                          moe_backend="hip", moe_router_dtype=torch.float32, router_alpha=0.01)
    torch.manual_seed(0)
    with torch.device("cuda"):
        moe = MoE(cfg, ffn=ffn)
    for p in moe.experts.parameters():
        p.data.normal_(0, p.shape[1] ** -0.5)
    return moe


@pytest.mark.parametrize("ffn", ["swiglu", "gelu"])
@pytest.mark.parametrize("how", ["forward", "pre", "override", "global"])
def test_what_hangs_on_the_experts_runs(ext, ffn, how):
    moe = _moe(ffn)
    e = moe.experts
    x = torch.randn(3, 4, 128, device="cuda").to(torch.bfloat16)
    before = moe.decode(x)
    seen = []

    def double(module, args, out):
        if module is e:
            seen.append(1)
            return 2 * out

    def zero(module, args):
        seen.append(1)
        return torch.zeros_like(args[0]), args[1]

    if how == "forward":
        handle = e.register_forward_hook(double)
    elif how == "pre":
        handle = e.register_forward_pre_hook(zero)
    elif how == "global":
        handle = torch.nn.modules.module.register_module_forward_hook(double)
    else:
        plain = e.forward
        e.forward = lambda *a: (seen.append(1), plain(*a) * 2)[1]
    try:
        got = moe.decode(x)
        assert len(seen) == 1
        with torch.no_grad():
            assert torch.equal(got, moe(x)[0])
    finally:
        if how == "override":
            del e.forward
        else:
            handle.remove()
    assert torch.equal(moe.decode(x), before)


@pytest.mark.parametrize("hooked", [False, True])
def test_sizes_do_not_depend_on_what_hangs(ext, hooked):
    moe = _moe("swiglu")
    if hooked:
        moe.experts.register_forward_hook(lambda module, args, out: out)
    dt = torch.bfloat16
    assert moe.decode(torch.zeros(1, 64, 128, device="cuda", dtype=dt)).shape == (1, 64, 128)
    assert moe.decode(torch.zeros(2, 0, 128, device="cuda", dtype=dt)).shape == (2, 0, 128)
    with pytest.raises(RuntimeError, match="at most"):
        moe.decode(torch.zeros(5, 13, 128, device="cuda", dtype=dt))

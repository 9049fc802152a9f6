"""Few-token layer, block norms and 8-bit checkpoints without a GPU: the 64-bit
oracle of the checkpoint format, and the refusals of the C ABI and the wrappers."""

from types import SimpleNamespace

import pytest
import torch

from nanotitan_amd import capi, moe_ops
from nanotitan_amd.layer import MoE, MoEBlock


def kept64(x):
    """(codes, exponent bytes) of a checkpoint of x (float64 rows), from the format's definition."""
    A, f = x.shape
    n = -(-f // 32)
    pad = torch.zeros(A, n * 32, dtype=torch.float64)
    pad[:, :f] = x
    blocks = pad.view(A, n, 32)
    most = blocks.abs().amax(-1)
    exp = torch.full((A, n), -127, dtype=torch.int64)
    for _ in range(400):  # the least integer with max < 127.5 units, from -127 up
        more = most >= 127.5 * torch.exp2(exp.double())
        if not bool(more.any()):
            break
        exp += more.to(torch.int64)
    units = blocks / torch.exp2(exp.double()).unsqueeze(-1)
    codes = torch.round(units).to(torch.int8).view(A, n * 32)[:, :f]
    return codes.contiguous(), (exp + 127).to(torch.uint8)


def held64(x, dtype=torch.float32):
    """The values that a checkpoint of x holds in ``dtype`` (none past its largest)."""
    codes, exps = kept64(x)
    unit = torch.exp2(exps.double() - 127.0).repeat_interleave(32, dim=1)[:, : x.shape[1]]
    most = torch.finfo(dtype).max
    return (codes.double() * unit).clamp(-most, most)


def test_oracle_of_the_checkpoint():
    x = torch.tensor([[127.0, 0.5, 1.5, -2.5], [127.5, 1.0, 3.0, -5.0], [0.0, 0.0, 0.0, 0.0],
                      [1.0, 1 / 128, -1 / 127, 0.25]], dtype=torch.float64)
    codes, exps = kept64(x)
    assert exps.tolist() == [[127], [128], [0], [121]]
    assert codes.tolist() == [[127, 0, 2, -2], [64, 0, 2, -2], [0, 0, 0, 0], [64, 0, -1, 16]]
    g = torch.randn(50, 100, dtype=torch.float64)
    err = (held64(g) - g).abs()
    unit = torch.exp2(kept64(g)[1].double() - 127).repeat_interleave(32, dim=1)[:, :100]
    assert bool((err <= unit / 2).all())


BF, F32 = capi.NT_BF16, capi.NT_F32
P = 4096  # a non-null address: none of these calls gets as far as using it


@pytest.mark.parametrize("fn,args,code", [
    ("nt_checkpoint8", (capi.NT_F64, P, 4, 8, P, P, None), capi.NT_ERR_DTYPE),
    ("nt_checkpoint8", (BF, P, -1, 8, P, P, None), capi.NT_ERR_INVALID_ARG),
    ("nt_checkpoint8", (BF, P, 4, 0, P, P, None), capi.NT_ERR_INVALID_ARG),
    ("nt_checkpoint8", (BF, P, 4, 8, None, P, None), capi.NT_ERR_INVALID_ARG),
    ("nt_checkpoint8", (BF, None, 0, 8, None, None, None), capi.NT_OK),
    ("nt_checkpoint8", (BF, P, 2**31, 8, P, P, None), capi.NT_ERR_TOO_LARGE),
    ("nt_checkpoint8", (BF, P, 2**31 - 1, 2**30, P, P, None), capi.NT_ERR_TOO_LARGE),
    ("nt_checkpoint8_decode", (7, P, P, 4, 8, P, None), capi.NT_ERR_DTYPE),
    ("nt_checkpoint8_decode", (BF, P, P, 4, 8, None, None), capi.NT_ERR_INVALID_ARG),
    ("nt_gelu_checkpoint8", (BF, P, 4, 8, P, P, None, None), capi.NT_ERR_INVALID_ARG),
    ("nt_gelu_backward8", (BF, P, P, P, 4, 8, None, None, None), capi.NT_ERR_INVALID_ARG),
    ("nt_swiglu_checkpoint8", (BF, P, P, 4, 8, P, P, P, P, None, None), capi.NT_ERR_INVALID_ARG),
    ("nt_swiglu_backward8", (BF, P, P, P, P, P, 4, 8, P, None, None, None),
     capi.NT_ERR_INVALID_ARG),
])
def test_checkpoint8_refusals(fn, args, code):
    assert getattr(capi.load(), fn)(*args) == code


def test_checkpoint8_blocks():
    blocks = capi.load().nt_checkpoint8_blocks
    assert [blocks(f) for f in (-1, 0, 1, 32, 33, 2048)] == [0, 0, 1, 1, 2, 64]


def _norm(**over):
    a = dict(x_dtype=BF, dtype=BF, param=BF, kind=0, x=P, y=P, w=P, b=None, gate=None, gate_cols=0,
             scale=None, scale_cols=0, w_next=P, b_next=None, eps=1e-6, T=4, d=8, h=P, n=P,
             stats=None, stream=None)
    a.update(over)
    return tuple(a.values())


@pytest.mark.parametrize("over,code", [
    (dict(dtype=capi.NT_F64, x_dtype=capi.NT_F64), capi.NT_ERR_DTYPE),
    (dict(x_dtype=BF, dtype=F32), capi.NT_ERR_DTYPE),  # a residual stream narrower than the block
    (dict(x_dtype=capi.NT_F16), capi.NT_ERR_DTYPE),
    (dict(param=capi.NT_F64), capi.NT_ERR_DTYPE),
    (dict(kind=2), capi.NT_ERR_INVALID_ARG),
    (dict(T=-1), capi.NT_ERR_INVALID_ARG),
    (dict(d=0), capi.NT_ERR_INVALID_ARG),
    (dict(d=16385), capi.NT_ERR_TOO_LARGE),
    (dict(T=2**31), capi.NT_ERR_TOO_LARGE),
    (dict(b=P), capi.NT_ERR_INVALID_ARG),  # rms norms have no bias
    (dict(kind=1, w=None, b=P), capi.NT_ERR_INVALID_ARG),
    (dict(kind=1, w_next=None, b_next=P), capi.NT_ERR_INVALID_ARG),
    (dict(gate=P, gate_cols=2), capi.NT_ERR_INVALID_ARG),
    (dict(scale=P, scale_cols=3), capi.NT_ERR_INVALID_ARG),
    (dict(y=None), capi.NT_ERR_INVALID_ARG),  # a weight for a branch that is not there
    (dict(y=None, w=None, w_next=None), capi.NT_ERR_INVALID_ARG),
    (dict(x=None), capi.NT_ERR_INVALID_ARG),
    (dict(h=None), capi.NT_ERR_INVALID_ARG),
    (dict(n=None), capi.NT_ERR_INVALID_ARG),
    (dict(T=0, x=None, h=None, n=None), capi.NT_OK),
])
def test_block_norm_refusals(over, code):
    assert capi.load().nt_block_norm(*_norm(**over)) == code


def _norm_grad(**over):
    a = dict(x_dtype=BF, dtype=BF, param=BF, kind=0, h=P, y=P, w=P, b=None, gate=None, gate_cols=0,
             scale=None, scale_cols=0, w_next=P, stats=P, dh=P, dn=P, T=4, d=8, dx=P, dy=P,
             dgate=None, dscale=None, dw=P, db=None, dw_next=P, db_next=None, ws=P, ws_bytes=1 << 20,
             stream=None)
    a.update(over)
    return tuple(a.values())


@pytest.mark.parametrize("over,code", [
    (dict(x_dtype=capi.NT_F64, dtype=capi.NT_F64), capi.NT_ERR_DTYPE),
    (dict(d=16385), capi.NT_ERR_TOO_LARGE),
    (dict(w_next=None), capi.NT_ERR_INVALID_ARG),  # dn without the norm it belongs to
    (dict(dgate=P), capi.NT_ERR_INVALID_ARG),
    (dict(dscale=P), capi.NT_ERR_INVALID_ARG),
    (dict(w=None), capi.NT_ERR_INVALID_ARG),
    (dict(y=None, w=None, dw=None), capi.NT_ERR_INVALID_ARG),
    (dict(db=P), capi.NT_ERR_INVALID_ARG),
    (dict(h=None), capi.NT_ERR_INVALID_ARG),
    (dict(stats=None), capi.NT_ERR_INVALID_ARG),
    (dict(ws=None), capi.NT_ERR_WORKSPACE),
    (dict(ws_bytes=4), capi.NT_ERR_WORKSPACE),
    (dict(T=0, dw=None, dw_next=None, h=None, ws=None), capi.NT_OK),
])
def test_block_norm_backward_refusals(over, code):
    assert capi.load().nt_block_norm_backward(*_norm_grad(**over)) == code


def _few(**over):
    a = dict(dtype=BF, x=P, router=P, logits=None, up=P, val=P, down=P, T=4, E=8, k=2, d=16, f=32,
             gates=P, topk=P, out=P, ws=P, ws_bytes=1 << 30, stream=None)
    a.update(over)
    return tuple(a.values())


@pytest.mark.parametrize("over,code", [
    (dict(dtype=capi.NT_F64), capi.NT_ERR_DTYPE),
    (dict(T=65), capi.NT_ERR_TOO_LARGE),
    (dict(T=-1), capi.NT_ERR_INVALID_ARG),
    (dict(E=1025), capi.NT_ERR_TOO_MANY_EXPERTS),
    (dict(E=64, k=33), capi.NT_ERR_INVALID_ARG),
    (dict(k=9), capi.NT_ERR_INVALID_ARG),
    (dict(k=0), capi.NT_ERR_INVALID_ARG),
    (dict(d=0), capi.NT_ERR_INVALID_ARG),
    (dict(f=0), capi.NT_ERR_INVALID_ARG),
    (dict(logits=P), capi.NT_ERR_INVALID_ARG),  # router and logits
    (dict(router=None), capi.NT_ERR_INVALID_ARG),  # neither
    (dict(x=None), capi.NT_ERR_INVALID_ARG),
    (dict(up=None), capi.NT_ERR_INVALID_ARG),
    (dict(down=None), capi.NT_ERR_INVALID_ARG),
    (dict(out=None), capi.NT_ERR_INVALID_ARG),
    (dict(ws=None), capi.NT_ERR_WORKSPACE),
    (dict(ws_bytes=16), capi.NT_ERR_WORKSPACE),
    (dict(ws=P + 4), capi.NT_ERR_WORKSPACE),
    (dict(T=0, x=None, ws=None), capi.NT_OK),
])
def test_few_tokens_refusals(over, code):
    assert capi.load().nt_moe_few_tokens(*_few(**over)) == code


def test_few_tokens_workspace():
    size = capi.load().nt_moe_few_tokens_workspace_bytes
    assert size(BF, 0, 8, 2, 16, 32) == 0 and size(BF, 65, 8, 2, 16, 32) == 0
    # at least the hidden rows and one partial sum a row
    assert size(BF, 16, 8, 2, 512, 2048) >= 32 * 2048 * 2 + 32 * 512 * 4


def test_wrappers_refuse_before_the_extension_runs():
    x = torch.zeros(4, 8)
    w = torch.ones(8)
    with pytest.raises(RuntimeError, match="norm kind"):
        moe_ops.pre_norm_fn(x, w, kind="batch")
    with pytest.raises(RuntimeError, match="gate must"):
        moe_ops.post_norm_fn(x, x, w, gate=torch.zeros(4, 2))
    with pytest.raises(RuntimeError, match="gate must"):
        moe_ops.post_norm_fn(x, x, w, gate=torch.zeros(1, 8))
    with pytest.raises(RuntimeError, match="one shape"):
        moe_ops.post_norm_fn(x, torch.zeros(8, 4), w)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        moe_ops.pre_norm_fn(x, w)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        moe_ops.checkpoint8(x)
    up, down = torch.zeros(2, 8, 16), torch.zeros(2, 16, 8)
    with pytest.raises(RuntimeError, match="weights are"):
        moe_ops.moe_few_tokens(x, (up,), 1, logits=torch.zeros(4, 2))
    with pytest.raises(RuntimeError, match="no backward"):
        moe_ops.moe_few_tokens(x.requires_grad_(), (up, down), 1, logits=torch.zeros(4, 2))
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU tensor"):
        moe_ops.moe_few_tokens(x, (up, down), 1, logits=torch.zeros(4, 2))


def _cfg(**over):
    return SimpleNamespace(**dict(num_experts=2, top_k=1, d_model=8, ffn_in=16, moe_backend="hip",
                                  dtype=torch.float32, router_alpha=0.01) | over)


def test_decode_refuses_foreign_experts():
    """Their weights may have another layout, or their forward another formula."""
    class Experts(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.W_up, self.W_down = torch.zeros(2, 8, 16), torch.zeros(2, 16, 8)

    moe = MoE(_cfg(), ffn="gelu")
    moe.experts = Experts()
    with pytest.raises(RuntimeError, match="not Experts"):
        moe.decode(torch.zeros(1, 2, 8))


@pytest.mark.parametrize("other", [dict(norm="layer"), dict(eps=1e-5)])
def test_block_refuses_to_take_another_norm_along(other):
    """One pass holds one kind of norm: the following block's would come out wrong."""
    block, following = MoEBlock(_cfg()), MoEBlock(_cfg(), **other)
    with pytest.raises(ValueError, match="following block's norm"):
        block(torch.zeros(1, 2, 8), following=following)
    with pytest.raises(ValueError, match="following block's norm"):
        block.decode(torch.zeros(1, 2, 8), following=following)

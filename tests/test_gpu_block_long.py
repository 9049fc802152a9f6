"""Tensors of more than 2^31 elements. Norms and 8-bit checkpoints: the last rows are those of
the same rows alone, bit for bit, and so are sums over rows of which all but these are zero."""

import pytest
import torch

from nanotitan_amd import moe_ops
from tests.test_gpu_block_norm import _grad64, _hat64

pytestmark = pytest.mark.gpu

D = 2048
ROWS = 2**31 // D + 300  # the last 300 rows lie past 2^31 elements
LAST = 257


def _rows(seed, rows=ROWS):
    x = torch.zeros(rows, D, dtype=torch.bfloat16, device="cuda")
    x[-LAST:].normal_(generator=torch.Generator(device="cuda").manual_seed(seed))
    return x


def test_checkpoints(ext):
    x, d = _rows(0), _rows(1)
    for call in (lambda v, _: moe_ops.checkpoint8(v),
                 lambda v, _: [moe_ops.checkpoint8_decode(*moe_ops.checkpoint8(v), v.dtype)],
                 lambda v, w: [moe_ops.swiglu8_fn(v, w), moe_ops.gelu8_fn(v)],
                 lambda v, w: list(ext.gelu_backward8(w, *moe_ops.checkpoint8(v), True))):
        with torch.no_grad():
            whole = [t[-LAST:].clone() for t in call(x, d)]
            for a, b in zip(whole, call(x[-LAST:].clone(), d[-LAST:].clone())):
                assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_norms(ext, kind):
    x, y, dh, dn = (_rows(i) for i in range(4))
    w = torch.linspace(0.5, 1.5, D, device="cuda")

    def run(*ts):
        leaf = [t.requires_grad_() for t in (ts[0], ts[1], w.clone())]
        h, n = moe_ops.post_norm_fn(*leaf, next_weight=w, kind=kind)
        grads = torch.autograd.grad([h, n], leaf, ts[2:])
        return [t.detach()[-LAST:].clone() for t in (h, n, *grads[:2])], grads[2].double()

    rows, dw = run(x, y, dh, dn)
    last = [t.detach()[-LAST:].clone() for t in (x, y, dh, dn)]
    alone, dw_alone = run(*last)
    for a, b in zip(rows, alone):
        assert torch.equal(a, b)
    # The same float32 products in two orders of at most 600 additions in a row each.
    _, y64, dh64, dn64 = (t.detach().double() for t in last)
    hhat, r = _hat64(rows[0].double(), kind)
    mag = ((dh64 + _grad64(dn64 * w, hhat, r, kind)) * _hat64(y64, kind)[0]).abs().sum(0)
    assert bool(((dw - dw_alone).abs() <= 2 * 600 * 2.0**-24 * mag).all())


def test_few_tokens(ext):
    """Experts whose weights lie past 2^31 elements, among others that no token chose."""
    T, E, d, f = 9, 38, 4096, 14336
    g = torch.Generator(device="cuda").manual_seed(9)
    up = torch.zeros(E, d, f, dtype=torch.bfloat16, device="cuda")
    down = torch.zeros(E, f, d, dtype=torch.bfloat16, device="cuda")
    assert (E - 1) * d * f > 2**31
    for e in (E - 2, E - 1):
        up[e].normal_(0, d**-0.5, generator=g)
        down[e].normal_(0, f**-0.5, generator=g)
    x = torch.empty(T, d, device="cuda").normal_(generator=g).to(torch.bfloat16)
    logits = torch.zeros(T, E, device="cuda")
    logits[:, E - 2], logits[:, E - 1] = 20.0, torch.linspace(18, 22, T, device="cuda")
    with torch.no_grad():
        out, gates, ids = moe_ops.moe_few_tokens(x, (up, down), 2, logits=logits)
    want = torch.zeros(T, d, dtype=torch.float64, device="cuda")
    for e in (E - 2, E - 1):
        h = torch.nn.functional.gelu(x.double() @ up[e].double())
        want += (gates * (ids == e)).sum(1, keepdim=True).double() * (h @ down[e].double())
    # the roundings of the hidden rows and of the output, half a step of the norm each, and
    # float32 sums of d and f terms in chains of d / 32 and f / 32 at most
    tol = torch.finfo(torch.bfloat16).eps + (d + f) / 32 * 2.0**-24
    assert bool(((out.double() - want).norm(dim=1) <= tol * want.norm(dim=1)).all())

"""Block norms (pre_norm_fn, post_norm_fn): forward and every gradient against
64 bits, over types, widths, gates, scales and what is left out."""

import pytest
import torch

from nanotitan_amd.moe_ops import post_norm_fn, pre_norm_fn

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 2.0**-24  # a float32 rounding
EPS = 1e-6


def _near(name, got, want, mag, ulps):
    """Half a step of got's type at want, and `ulps` float32 roundings of sums of size mag."""
    dt = got.dtype
    got = got.detach().cpu().double()
    tol = torch.finfo(dt).eps / 2 * want.abs() * (1 + 2.0**-8) + ulps * U * mag
    if dt == torch.float16:
        tol = tol + 2.0**-25
    off = (got - want).abs() - tol
    assert bool((off <= 0).all()), (name, float(off.max()))


def _hat64(v, kind):
    m = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    r = 1.0 / torch.sqrt(((v - m) ** 2).mean(-1, keepdim=True) + EPS)
    return (v - m) * r, r


def _grad64(u, hat, r, kind):
    g = u - hat * (u * hat).mean(-1, keepdim=True)
    return r * (g - u.mean(-1, keepdim=True) if kind == "layer" else g)


def _case(T, d, x_dt, dt, p_dt, kind, gate, scale, post, nxt, seed=0):
    g = torch.Generator().manual_seed(seed)

    def t(*shape, std=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g) * std + mean).to(dtype)

    layer = kind == "layer"
    return dict(
        x=t(T, d, dtype=x_dt), y=t(T, d, std=0.5, mean=0.2),
        w=t(d, std=0.3, mean=1.0, dtype=p_dt) if post else None,
        b=t(d, std=0.3, dtype=p_dt) if post and layer else None,
        gate={"none": None, "token": t(T, 1), "full": t(T, d)}[gate],
        scale={"none": None, "one": t(1, dtype=p_dt), "channel": t(d, dtype=p_dt)}[scale],
        wn=t(d, std=0.3, mean=1.0, dtype=p_dt) if nxt else None,
        bn=t(d, std=0.3, dtype=p_dt) if nxt and layer else None,
        dh=t(T, d, dtype=x_dt), dn=t(T, d) if nxt else None)


def _run(c, kind, grad=True, dh=True, dn=True):
    names = ["x", "y", "w", "b", "gate", "scale", "wn", "bn"]
    leaf = {n: None if c[n] is None else c[n].cuda().requires_grad_(grad) for n in names}
    out = post_norm_fn(leaf["x"], leaf["y"], leaf["w"], leaf["b"], gate=leaf["gate"],
                       scale=leaf["scale"], next_weight=leaf["wn"], next_bias=leaf["bn"],
                       kind=kind, eps=EPS)
    h, n = out if c["wn"] is not None else (out, None)
    if not grad:
        return h, n, {}
    outs, gs = [], []
    if dh:
        outs.append(h), gs.append(c["dh"].cuda())
    if n is not None and dn:
        outs.append(n), gs.append(c["dn"].cuda())
    live = [k for k in names if leaf[k] is not None]
    grads = torch.autograd.grad(outs, [leaf[k] for k in live], gs, allow_unused=True)
    return h, n, dict(zip(live, grads))


def _check(c, kind, got_h, got_n, grads, dh=True, dn=True):
    z = {k: None if v is None else v.double() for k, v in c.items()}
    x, y = z["x"], z["y"]
    T, d = x.shape
    one = torch.ones(1, dtype=torch.float64)
    w, wn = (z[k] if z[k] is not None else one for k in ("w", "wn"))
    b, bn = (z[k] if z[k] is not None else 0 * one for k in ("b", "bn"))
    gate, scale = (z[k] if z[k] is not None else one for k in ("gate", "scale"))
    post = z["w"] is not None
    yhat, ry = _hat64(y, kind) if post else (y, torch.ones(T, 1, dtype=torch.float64))
    p = yhat * w + b
    # a row's sums are at most 11 additions deep a lane and in the tree, and the centred
    # value loses the size of what was centred
    spread = (y.abs() + y.abs().mean(-1, keepdim=True)) * ry if post else y.abs()
    pmag = spread * w.abs() + (b.abs() if torch.is_tensor(b) else 0)
    _near("h", got_h, x + scale * gate * p, x.abs() + (scale * gate).abs() * pmag, 40)
    h = got_h.detach().cpu().double()  # the norm and the gradients are of h as it is held
    hhat, rh = _hat64(h, kind)
    hspread = (h.abs() + h.abs().mean(-1, keepdim=True)) * rh
    if got_n is not None:
        _near("n", got_n, hhat * wn + bn, hspread * wn.abs() + bn.abs(), 40)
    if not grads:
        return
    D = z["dh"] if dh else torch.zeros_like(x)
    Dmag = D.abs()
    if got_n is not None and dn:
        u = z["dn"] * wn
        D = D + _grad64(u, hhat, rh, kind)
        Dmag = Dmag + rh * (u.abs() + u.abs().mean(-1, keepdim=True)
                            + hspread * (u.abs() * hspread).mean(-1, keepdim=True))
    dp = D * gate * scale
    dpmag = Dmag * (gate * scale).abs()
    u, umag = dp * w, dpmag * w.abs()
    dy = _grad64(u, yhat, ry, kind) if post else u
    dymag = ry * (umag + umag.mean(-1, keepdim=True)
                  + spread * (umag * spread).mean(-1, keepdim=True)) if post else umag
    dg, dgmag = D * scale * p, Dmag * scale.abs() * pmag
    ds, dsmag = D * gate * p, Dmag * gate.abs() * pmag
    want = {"x": (D, Dmag), "y": (dy, dymag),
            "w": ((dp * yhat).sum(0), (dpmag * spread).sum(0)), "b": (dp.sum(0), dpmag.sum(0)),
            "gate": (dg, dgmag), "scale": (ds.sum(0), dsmag.sum(0))}
    if z["gate"] is not None and z["gate"].shape[1] == 1:
        want["gate"] = (dg.sum(-1, keepdim=True), dgmag.sum(-1, keepdim=True))
    if z["scale"] is not None and z["scale"].numel() == 1:
        want["scale"] = (ds.sum().view(1), dsmag.sum().view(1))
    if got_n is not None:
        gn = z["dn"] if dn else torch.zeros_like(x)
        want["wn"] = ((gn * hhat).sum(0), (gn.abs() * hspread).sum(0))
        want["bn"] = (gn.sum(0), gn.abs().sum(0))
    for k, g in grads.items():
        if g is None:
            assert float(want[k][0].abs().max()) == 0.0, k
            continue
        assert g.dtype == c[k].dtype and g.shape == c[k].shape
        # sums over the tokens: at most 512 additions in a row (a workgroup's rows, then
        # every fourth workgroup)
        _near("d" + k, g, want[k][0], want[k][1], 100 if k in ("x", "y", "gate") else 600)


WIDTHS = [1, 7, 64, 128, 130, 300, 512, 513, 1000, 1024, 2048, 2056, 4096, 5000, 8192, 8200, 16384]


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("d", WIDTHS)
def test_widths(ext, kind, d):
    for dtype in TYPES.values():
        c = _case(9, d, dtype, dtype, dtype, kind, "full", "channel", True, True, seed=d)
        _check(c, kind, *_run(c, kind))


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 1025, 4100])
@pytest.mark.parametrize("d", [96, 300, 1024])
def test_row_counts(ext, T, d):
    c = _case(T, d, torch.bfloat16, torch.bfloat16, torch.float32, "layer", "token", "one", True,
              True, seed=T)
    _check(c, "layer", *_run(c, "layer"))


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "token", "full"])
@pytest.mark.parametrize("scale", ["none", "one", "channel"])
@pytest.mark.parametrize("post,nxt", [(True, True), (True, False), (False, True), (False, False)])
def test_what_is_left_out(ext, kind, gate, scale, post, nxt):
    for x_dt, dt, p_dt in ((torch.bfloat16,) * 3, (torch.float32, torch.float16, torch.float32),
                           (torch.float32, torch.bfloat16, torch.bfloat16)):
        for d in (200, 2048):
            c = _case(21, d, x_dt, dt, p_dt, kind, gate, scale, post, nxt)
            h, n, grads = _run(c, kind)
            _check(c, kind, h, n, grads)
            h2, n2, _ = _run(c, kind, grad=False)
            assert torch.equal(h, h2) and (n is None or torch.equal(n, n2))


def test_any_one_input_alone(ext):
    """Frozen inputs get no gradient, and the others the bits that they get together."""
    c = _case(40, 264, torch.bfloat16, torch.bfloat16, torch.float32, "layer", "token", "channel",
              True, True)
    _, _, full = _run(c, "layer")
    names = ["x", "y", "w", "b", "gate", "scale", "wn", "bn"]
    for alone in names:
        leaf = {n: c[n].cuda().requires_grad_(n == alone) for n in names}
        h, n = post_norm_fn(leaf["x"], leaf["y"], leaf["w"], leaf["b"], gate=leaf["gate"],
                            scale=leaf["scale"], next_weight=leaf["wn"], next_bias=leaf["bn"],
                            kind="layer", eps=EPS)
        outs = [(h, c["dh"].cuda())] if alone not in ("wn", "bn") else []
        outs.append((n, c["dn"].cuda()))
        (g,) = torch.autograd.grad([o for o, _ in outs], [leaf[alone]], [g for _, g in outs])
        assert torch.equal(g, full[alone]), alone
        assert all(v.grad is None for v in leaf.values())


@pytest.mark.parametrize("dh,dn", [(True, False), (False, True)])
@pytest.mark.parametrize("d", [72, 1536])
def test_only_one_output_used(ext, dh, dn, d):
    c = _case(33, d, torch.float32, torch.float32, torch.float32, "layer", "full", "channel",
              True, True)
    _check(c, "layer", *_run(c, "layer", dh=dh, dn=dn), dh=dh, dn=dn)


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("x_dt,dt", [("fp32", "fp32"), ("fp32", "bf16"), ("fp16", "fp16")])
@pytest.mark.parametrize("shape", [(5, 40), (3, 4, 700), (2, 3, 2, 4096)])
def test_pre_norm(ext, kind, x_dt, dt, shape):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(*shape, generator=g).to(TYPES[x_dt])
    w = (torch.randn(shape[-1], generator=g) + 1).to(TYPES[dt])
    b = torch.randn(shape[-1], generator=g).to(TYPES[dt]) if kind == "layer" else None
    dn = torch.randn(*shape, generator=g).to(TYPES[dt])
    leaf = [None if t is None else t.cuda().requires_grad_() for t in (x, w, b)]
    n = pre_norm_fn(*leaf, kind=kind, eps=EPS, dtype=TYPES[dt])
    assert n.shape == x.shape and n.dtype == TYPES[dt]
    grads = torch.autograd.grad(n, [t for t in leaf if t is not None], dn.cuda())
    x64, w64, dn64 = (t.double().reshape(-1, shape[-1]) for t in (x, w.expand(shape), dn))
    hat, r = _hat64(x64, kind)
    spread = (x64.abs() + x64.abs().mean(-1, keepdim=True)) * r
    b64 = 0 * w64 if b is None else b.double()
    flat = lambda t: t.reshape(-1, shape[-1]) if t.dim() > 1 else t  # noqa: E731
    _near("n", flat(n), hat * w64 + b64, spread * w64.abs() + b64.abs(), 40)
    u = dn64 * w64
    mag = r * (u.abs() + u.abs().mean(-1, keepdim=True)
               + spread * (u.abs() * spread).mean(-1, keepdim=True))
    _near("dx", flat(grads[0]), _grad64(u, hat, r, kind), mag, 100)
    _near("dw", grads[1], (dn64 * hat).sum(0), (dn64.abs() * spread).sum(0), 600)
    if b is not None:
        _near("db", grads[2], dn64.sum(0), dn64.abs().sum(0), 600)


def test_against_differences(ext):
    """Directional derivatives of the float32 forward, step 2^-7, in every input at once."""
    c = _case(12, 160, torch.float32, torch.float32, torch.float32, "layer", "full", "channel",
              True, True, seed=5)
    _, _, grads = _run(c, "layer")

    def value(at):
        h, n, _ = _run({**c, **at}, "layer", grad=False)
        return (h.cpu().double() * c["dh"].double()).sum() + (
            n.cpu().double() * c["dn"].double()).sum()

    g = torch.Generator().manual_seed(6)
    for k, grad in grads.items():
        v = torch.randn(c[k].shape, generator=g)
        v = v / v.norm()
        e = 2.0**-7
        diff = (value({k: c[k] + e * v}) - value({k: c[k] - e * v})) / (2 * e)
        want = (grad.cpu().double() * v.double()).sum()
        # e^2 of the third derivatives (of the order of the gradient), and the float32
        # roundings of 2 x 1920 outputs of order one over 2 e
        tol = 2.0**-10 * float(grad.double().norm()) + 1920**0.5 * 8 * U / e
        assert abs(float(diff - want)) <= tol, (k, float(diff), float(want))


def test_rows_that_hold_nothing_or_too_much(ext):
    """A zero row, a constant row, an infinity and a NaN touch their own rows only."""
    d = 320
    x = torch.randn(6, d)
    y = torch.randn(6, d)
    y[0] = 0
    y[1] = 3.0
    y[2, 5] = float("inf")
    y[3, 7] = float("nan")
    w = torch.ones(d)
    for kind in ("rms", "layer"):
        h, n = post_norm_fn(x.cuda(), y.cuda(), w.cuda(), kind=kind, next_weight=w.cuda(), eps=EPS)
        h, n = h.cpu(), n.cpu()
        assert torch.equal(h[0], x[0])
        if kind == "layer":  # the mean of a constant row is off by a few roundings of 3
            assert float((h[1] - x[1]).abs().max()) <= 40 * U * 3 / EPS**0.5
        assert bool(h[2].isnan().any()) and bool(h[3].isnan().all() if kind == "rms"
                                                 else h[3].isnan().any())
        for r in (0, 1, 4, 5):
            assert bool(h[r].isfinite().all()) and bool(n[r].isfinite().all())


def test_no_rows(ext):
    w = torch.ones(64, device="cuda", requires_grad=True)
    s = torch.ones(1, device="cuda", requires_grad=True)
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    h, n = post_norm_fn(x, x, w, scale=s, next_weight=w)
    assert h.shape == n.shape == (0, 64)
    dw, ds = torch.autograd.grad(h.sum() + n.sum(), [w, s])
    assert float(dw.abs().max()) == 0.0 and float(ds) == 0.0


def test_any_address_layout_and_shared_inputs(ext):
    d, T = 77, 30
    dt = torch.bfloat16
    buf = torch.randn(T * d + 1).to(dt).cuda()
    x = buf[1:].view(T, d)
    w = torch.randn(d + 1).to(dt).cuda()[1:]
    ref = post_norm_fn(x.clone(), x.clone(), w.clone(), next_weight=w.clone())
    got = post_norm_fn(x, x, w, next_weight=w)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    t = torch.randn(d, T).to(dt).cuda().t()  # strided rows
    assert torch.equal(pre_norm_fn(t, w), pre_norm_fn(t.contiguous(), w))
    # x as its own branch and one weight twice: the gradients add up
    xl, wl = torch.randn(T, d, device="cuda").requires_grad_(), w.float().requires_grad_()
    h, n = post_norm_fn(xl, xl, wl, next_weight=wl)
    dx, dw = torch.autograd.grad([h, n], [xl, wl], [torch.ones_like(h), torch.ones_like(n)])
    parts = [xl.detach().requires_grad_() for _ in range(2)] + [
        wl.detach().requires_grad_() for _ in range(2)]
    h2, n2 = post_norm_fn(parts[0], parts[1], parts[2], next_weight=parts[3])
    g = torch.autograd.grad([h2, n2], parts, [torch.ones_like(h), torch.ones_like(n)])
    assert torch.equal(dx, g[0] + g[1]) and torch.equal(dw, g[2] + g[3])


def test_repeatable_in_a_graph_and_on_another_stream(ext):
    c = _case(700, 384, torch.bfloat16, torch.bfloat16, torch.float32, "layer", "full", "one",
              True, True)
    leaf = {k: None if v is None else v.cuda().requires_grad_(k not in ("dh", "dn"))
            for k, v in c.items()}
    ins = [leaf[k] for k in ("x", "y", "w", "b", "gate", "scale", "wn", "bn")]

    def step():
        h, n = post_norm_fn(leaf["x"], leaf["y"], leaf["w"], leaf["b"], gate=leaf["gate"],
                            scale=leaf["scale"], next_weight=leaf["wn"], next_bias=leaf["bn"],
                            kind="layer")
        grads = torch.autograd.grad([h, n], ins, [leaf["dh"], leaf["dn"]])
        # no eager graph of the leaves may live while one is captured
        return [h.detach(), n.detach(), *grads]

    first = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, on_side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (1, 2, 3):
        with torch.no_grad():
            leaf["y"].copy_(torch.randn(700, 384, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_refusals(ext):
    x = torch.randn(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    h16 = x.half()
    for bad in (lambda: pre_norm_fn(x, w, w),  # rms norms have no bias
                lambda: pre_norm_fn(x, w[:32]),
                lambda: pre_norm_fn(x, w.double()),
                lambda: pre_norm_fn(h16, w, dtype=torch.float32),
                lambda: pre_norm_fn(x.double(), w),
                lambda: pre_norm_fn(x, w.cpu()),
                lambda: post_norm_fn(h16, x, w),  # a stream narrower than the block's type
                lambda: post_norm_fn(x, x, w, scale=w[:2]),
                lambda: post_norm_fn(x, x, w, scale=w.half()),  # mixed parameter types
                lambda: post_norm_fn(x, x, w, gate=h16),
                lambda: post_norm_fn(x, x, None, w),  # a bias without its norm
                lambda: pre_norm_fn(torch.randn(2, 16385, device="cuda"),
                                    torch.ones(16385, device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()
    xl = x.requires_grad_()
    (g,) = torch.autograd.grad(pre_norm_fn(xl, w).square().sum(), xl, create_graph=True)
    with pytest.raises(RuntimeError):  # once differentiable
        torch.autograd.grad(g.sum(), xl)

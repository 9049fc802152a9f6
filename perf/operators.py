"""The operators of an MoE block around and beside its expert path, as measurable cases.

A case is one pass through one operator's public entry point, described by
plain values:

* ``op="few"``: ``moe_few_tokens``, a whole MoE layer for the few tokens of a
  decode step (router or logits, top-k, experts, gate-weighted sum).
* ``op="norm"``: ``post_norm_fn``, the norm after a block with its gate and
  residual scale, the residual sum, and the norm before the next block;
  ``step``: ``"infer"`` (forward) or ``"train"`` (forward and every gradient).
* ``op="act8"``: ``swiglu8_fn`` / ``gelu8_fn``, an expert FFN's activation that
  keeps its inputs in 8 bits for the backward; forward and gradients.
* ``op="store8"``: ``checkpoint8`` and ``checkpoint8_decode``, packed token rows
  kept in 8 bits and brought back.

With ``own`` false the same is computed by elementary torch operations in
32 bits.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
BLOCK = 32


def _few(name, dtype, ffn, T, d, f, E, k, router):
    return dict(name=name, op="few", dtype=dtype, ffn=ffn, T=T, d=d, f=f, E=E, k=k, router=router)


def _norm(name, step, dtype, kind, T, d, gate, scale):
    return dict(name=name, op="norm", step=step, dtype=dtype, kind=kind, T=T, d=d, gate=gate,
                scale=scale)


def _act8(name, dtype, ffn, A, f):
    return dict(name=name, op="act8", dtype=dtype, ffn=ffn, A=A, f=f)


def listed():
    return [
        # One sequence decoding through the small training configuration's layer: latency.
        _few("few_one", "bf16", "swiglu", 1, 512, 2048, 16, 2, True),
        # The same layer in full precision, unrounded 8 d / 3 experts, a few sequences.
        _few("few_fp32_odd", "fp32", "swiglu", 7, 512, 1365, 8, 2, True),
        # Many narrow experts, one to four rows each, gates from the program's own router.
        _few("few_fine", "fp16", "gelu", 33, 2048, 768, 128, 8, False),
        # A serving batch through a large-hidden layer: all experts' weights for 16 tokens.
        _few("few_wide", "bf16", "swiglu", 16, 4096, 14336, 8, 2, True),
        # A full batch of decoding sequences through the same layer.
        _few("few_full", "bf16", "swiglu", 64, 4096, 14336, 8, 2, True),
        # The norms of a decode step at the large-hidden width: one short launch.
        _norm("norm_decode", "infer", "bf16", "rms", 16, 4096, "none", "none"),
        # Full-precision LayerNorm blocks of an odd width, a learned scale per channel.
        _norm("norm_fp32_odd", "train", "fp32", "layer", 5003, 300, "none", "channel"),
        # The repository's training shape with an elementwise gate and one residual scale.
        _norm("norm_base", "train", "bf16", "rms", 40 * 768, 512, "full", "one"),
        # The large-hidden training shape with a gate per token.
        _norm("norm_wide", "train", "bf16", "rms", 16384, 4096, "token", "channel"),
        # The GELU experts' hidden rows at an odd width.
        _act8("gelu8_odd", "fp16", "gelu", 10007, 1365),
        # SwiGLU experts at the training shape: top-2 of 40 x 768 tokens.
        _act8("swiglu8_base", "bf16", "swiglu", 2 * 40 * 768, 2048),
        # The packed rows of fine-grained experts, the input that their dW needs again.
        dict(name="store8_rows", op="store8", dtype="bf16", A=8 * 40 * 768, f=512),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case of the listed ones' ranges; rows and widths are any number."""
    kind = rng.choice(["few_small", "few_fine", "few_wide", "norm_infer", "norm_train", "act8",
                       "store8"])
    half = rng.choice(["bf16", "fp16"])
    any_type = rng.choice(["bf16", "fp16", "fp32"])
    ffn = rng.choice(["swiglu", "gelu"])
    if kind == "few_small":
        d = rng.choice([128, 256, 300, 512, 768, 1024])
        c = _few("", any_type, ffn, _log_int(rng, 1, 64), d, rng.choice([8 * d // 3, 4 * d]),
                 rng.choice([4, 8, 16, 32]), rng.choice([1, 2, 4]), rng.random() < 0.5)
    elif kind == "few_fine":
        c = _few("", half, ffn, _log_int(rng, 1, 64), 2048, 768, rng.choice([64, 128]), 8,
                 rng.random() < 0.5)
    elif kind == "few_wide":
        c = _few("", half, ffn, _log_int(rng, 1, 60), 4096, 14336, 8, 2, True)
    elif kind.startswith("norm"):
        step = kind[len("norm_"):]
        d = rng.choice([rng.randint(64, 1024), 8 * rng.randint(8, 1024), 512, 2048, 4096, 8192])
        rows = _log_int(rng, 1, 256) if step == "infer" else _log_int(
            rng, 256, max(257, min(32768, 2**26 // d)))
        c = _norm("", step, any_type, rng.choice(["rms", "layer"]), rows, d,
                  rng.choice(["none", "token", "full"]), rng.choice(["none", "one", "channel"]))
    elif kind == "act8":
        f = rng.choice([rng.randint(64, 3000), 768, 1365, 2048])
        c = _act8("", any_type, ffn, _log_int(rng, 64, 2**26 // f), f)
    else:
        f = rng.choice([rng.randint(64, 2048), 512, 2048])
        c = dict(name="", op="store8", dtype=any_type, A=_log_int(rng, 64, 2**26 // f), f=f)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs


def _bias(case):
    return case["kind"] == "layer"


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, mean=0.0, dt=dtype):
        return torch.empty(*shape, dtype=dt, device="cuda").normal_(mean, std, generator=g)

    s = SimpleNamespace(case=case, dtype=dtype)
    if case["op"] == "few":
        T, d, f, E = (case[n] for n in ("T", "d", "f", "E"))
        s.x = randn(T, d)
        s.router = randn(E, d, std=d ** -0.5, dt=torch.float32) if case["router"] else None
        s.logits = None if case["router"] else randn(T, E, dt=torch.float32)
        # trained weights' scale: activations of unit order through both layers
        up = [randn(E, d, f, std=d ** -0.5) for _ in range(2 if case["ffn"] == "swiglu" else 1)]
        s.weights = (*up, randn(E, f, d, std=f ** -0.5))
        return s
    if case["op"] == "norm":
        T, d = case["T"], case["d"]
        s.x, s.y = randn(T, d), randn(T, d, std=0.5, mean=0.1)
        s.w, s.w_next = randn(d, std=0.2, mean=1.0), randn(d, std=0.2, mean=1.0)
        s.b, s.b_next = (randn(d, std=0.1), randn(d, std=0.1)) if _bias(case) else (None, None)
        s.gate = {"none": None, "token": (T, 1), "full": (T, d)}[case["gate"]]
        if s.gate is not None:
            s.gate = torch.sigmoid(randn(*s.gate))
        s.scale = {"none": None, "one": (1,), "channel": (d,)}[case["scale"]]
        if s.scale is not None:
            s.scale = randn(*s.scale, std=0.05, mean=0.3)
        if case["step"] == "train":
            s.dh, s.dn = randn(T, d), randn(T, d)
        return s
    A, f = case["A"], case["f"]
    s.x = randn(A, f)
    if case["op"] == "act8":
        s.value = randn(A, f) if case["ffn"] == "swiglu" else None
        s.dout = randn(A, f)
    return s


# --------------------------------------------------------------------- run


def run(s):
    op = s.case["op"]
    if op == "few":
        return _run_few(s)
    if op == "norm":
        return _run_norm(s)
    if op == "act8":
        return _run_act8(s)
    return _run_store8(s)


def _run_few(s):
    k = s.case["k"]
    if own:
        from nanotitan_amd.moe_ops import moe_few_tokens

        with torch.no_grad():
            out, gates, ids = moe_few_tokens(s.x, s.weights, k, router_weight=s.router,
                                             logits=s.logits)
        return [out, gates, ids]
    x = s.x.float()
    logits = s.logits if s.router is None else x @ s.router.t()
    # stable: equal logits go to the lower expert
    ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :k]
    top = logits.gather(1, ids)
    p = torch.exp(top - top[:, :1])
    gates = p / p.sum(-1, keepdim=True)
    # every expert on every token, weighted by a gate that is zero where it was not chosen
    dense = torch.zeros_like(logits).scatter_(1, ids, gates)
    h = torch.matmul(x, s.weights[0].float())  # [E, T, f]
    if s.case["ffn"] == "swiglu":
        h = h / (1.0 + torch.exp(-h)) * torch.matmul(x, s.weights[1].float())
    else:
        h = 0.5 * h * (1.0 + torch.erf(h * 0.5 ** 0.5))
    y = torch.matmul(h, s.weights[-1].float())
    out = (dense.t().unsqueeze(-1) * y).sum(0)
    return [out.to(s.dtype), gates, ids.to(torch.int32)]


def _hat(v, kind):
    """(v normalised, 1 / its deviation), rows in 32 bits."""
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    r = torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return v * r, r


def _hat_grad(u, hat, r, kind):
    g = u - hat * (u * hat).mean(-1, keepdim=True)
    if kind == "layer":
        g = g - u.mean(-1, keepdim=True)
    return g * r


def _run_norm(s):
    kind, train = s.case["kind"], s.case["step"] == "train"
    named = [("x", s.x), ("y", s.y), ("w", s.w), ("b", s.b), ("gate", s.gate),
             ("scale", s.scale), ("w_next", s.w_next), ("b_next", s.b_next)]
    if own:
        from nanotitan_amd.moe_ops import post_norm_fn

        a = {n: None if v is None else v.detach().requires_grad_(train) for n, v in named}
        h, n = post_norm_fn(a["x"], a["y"], a["w"], a["b"], gate=a["gate"], scale=a["scale"],
                            next_weight=a["w_next"], next_bias=a["b_next"], kind=kind, eps=EPS)
        if not train:
            return [h, n]
        return [h, n, *torch.autograd.grad([h, n], [v for v in a.values() if v is not None],
                                           [s.dh, s.dn])]
    x, y, w, b, gate, scale, w_next, b_next = (None if v is None else v.float() for _, v in named)
    yhat, ry = _hat(y, kind)
    p = yhat * w if b is None else yhat * w + b
    m = 1.0 if gate is None else gate
    sc = 1.0 if scale is None else scale
    h = (x + sc * m * p).to(s.dtype)
    hhat, rh = _hat(h.float(), kind)  # the next norm takes the residual stream as it is held
    n = hhat * w_next if b_next is None else hhat * w_next + b_next
    outs = [h, n]
    if train:
        dn = s.dn.float()
        D = s.dh.float() + _hat_grad(dn * w_next, hhat, rh, kind)
        dp = D * m * sc
        grads = [D, _hat_grad(dp * w, yhat, ry, kind), (dp * yhat).sum(0)]
        if b is not None:
            grads.append(dp.sum(0))
        if gate is not None:
            dg = D * sc * p
            grads.append(dg.sum(-1, keepdim=True) if gate.shape[1] == 1 else dg)
        if scale is not None:
            ds = D * m * p
            grads.append(ds.sum(0) if scale.numel() > 1 else ds.double().sum().reshape(1))
        grads.append((dn * hhat).sum(0))
        if b_next is not None:
            grads.append(dn.sum(0))
        outs += grads
    return [o.to(s.dtype) for o in outs]


def _through8(v):
    """v as its 8-bit checkpoint holds it: blocks of 32 columns share a power of two."""
    A, f = v.shape
    pad = -f % BLOCK
    x = torch.nn.functional.pad(v.float(), (0, pad)).view(A, -1, BLOCK)
    mant, ex = torch.frexp(x.abs().amax(-1, keepdim=True))  # mant in [1/2, 1)
    # the least power with max < 127.5 units
    ex = (ex - 7 + (mant >= 127.5 / 128).to(torch.int32)).clamp(min=-127)
    x = torch.ldexp(torch.round(torch.ldexp(x, -ex)), ex)
    return x.view(A, f + pad)[:, :f]


def _run_act8(s):
    swiglu = s.case["ffn"] == "swiglu"
    if own:
        from nanotitan_amd.moe_ops import gelu8_fn, swiglu8_fn

        a = [v.detach().requires_grad_() for v in ([s.x, s.value] if swiglu else [s.x])]
        out = swiglu8_fn(*a) if swiglu else gelu8_fn(*a)
        return [out, *torch.autograd.grad(out, a, s.dout)]
    x, dout = s.x.float(), s.dout.float()
    if swiglu:
        out = x / (1.0 + torch.exp(-x)) * s.value.float()
        g, v = _through8(s.x), _through8(s.value)
        sg = 1.0 / (1.0 + torch.exp(-g))
        outs = [out, dout * v * sg * (1.0 + g * (1.0 - sg)), dout * g * sg]
    else:
        out = 0.5 * x * (1.0 + torch.erf(x * 0.5 ** 0.5))
        h = _through8(s.x)
        slope = 0.5 * (1.0 + torch.erf(h * 0.5 ** 0.5)) + h * torch.exp(-0.5 * h * h) / math.sqrt(
            2.0 * math.pi)
        outs = [out, dout * slope]
    return [o.to(s.dtype) for o in outs]


def _run_store8(s):
    if own:
        from nanotitan_amd.moe_ops import checkpoint8, checkpoint8_decode

        codes, exps = checkpoint8(s.x)
        return checkpoint8_decode(codes, exps, s.dtype)
    return _through8(s.x).to(s.dtype)


# -------------------------------------------------------------------- work


def work(case):
    c = case
    b = torch.finfo(DTYPES[c["dtype"]]).bits // 8
    if c["op"] == "few":
        T, d, f, E, k = (c[n] for n in ("T", "d", "f", "E", "k"))
        mats = 3 if c["ffn"] == "swiglu" else 2
        # the chosen experts' weights, expected under uniform routing
        live = E * (1.0 - (1.0 - k / E) ** T)
        router = E * d * 4 if c["router"] else T * E * 4
        return {"bytes": int(mats * d * f * b * live + 2 * T * d * b + router + 8 * T * k),
                "flops": 2 * mats * T * k * d * f}
    if c["op"] == "norm":
        T, d = c["T"], c["d"]
        full = c["gate"] == "full"
        tensors = 4 + full  # x, y, gate in; h, n out
        if c["step"] == "train":
            tensors += 4 + full  # dh, dn in; dx, dy, dgate out
        return {"bytes": tensors * T * d * b, "flops": (40 if c["step"] == "train" else 12) * T * d}
    n = c["A"] * c["f"]
    code = 1 + 1 / BLOCK  # written once, read once
    if c["op"] == "act8":
        kept = 2 if c["ffn"] == "swiglu" else 1
        # in: the activation's inputs and the output's gradient; out: output, gradients
        return {"bytes": int(n * ((2 + 2 * kept) * b + 2 * kept * code)), "flops": 30 * n}
    return {"bytes": int(n * (2 * b + 2 * code)), "flops": 6 * n}


# ------------------------------------------------------------------- exact


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "few":
        return _exact_few(s)
    if op == "norm":
        return _exact_norm(s)
    x = s.x.double()
    if op == "store8":
        return _held64(x)
    if case["ffn"] == "swiglu":
        at = [_held64(x).requires_grad_(), _held64(s.value.double()).requires_grad_()]
        fn = lambda g, v: torch.nn.functional.silu(g) * v  # noqa: E731
        out = fn(x, s.value.double())
    else:
        at = [_held64(x).requires_grad_()]
        fn = torch.nn.functional.gelu
        out = fn(x)
    return [out, *torch.autograd.grad(fn(*at), at, s.dout.double())]


def _held64(x):
    """Every value to the nearest multiple (ties to even) of its block's power of two."""
    A, f = x.shape
    col = torch.arange(f, device=x.device) // BLOCK
    most = torch.zeros(A, int(col[-1]) + 1, dtype=torch.float64, device=x.device)
    most.scatter_reduce_(1, col.expand(A, f), x.abs(), "amax")
    ex = torch.floor(torch.log2(most / 127.5)) + 1.0
    unit = torch.exp2(ex.clamp(min=-127.0))[:, col]
    return torch.round(x / unit) * unit


def _exact_few(s):
    c = s.case
    x = s.x.double()
    logits = s.logits.double() if s.router is None else x @ s.router.double().t()
    ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :c["k"]]
    gates = logits.gather(1, ids).softmax(-1)
    out = torch.zeros_like(x)
    for e in torch.unique(ids).tolist():
        t, j = torch.nonzero(ids == e, as_tuple=True)
        w = [m[e].double() for m in s.weights]
        h = x[t] @ w[0]
        h = torch.nn.functional.silu(h) * (x[t] @ w[1]) if len(w) == 3 else (
            torch.nn.functional.gelu(h))
        out.index_add_(0, t, gates[t, j].unsqueeze(1) * (h @ w[-1]))
    return [out, gates, ids.to(torch.int32)]


def _norm64(v, w, b, kind):
    if kind == "layer":
        return torch.nn.functional.layer_norm(v, v.shape[-1:], w, b, EPS)
    return v / (v.square().mean(-1, keepdim=True) + EPS).sqrt() * w


def _exact_norm(s):
    kind, train = s.case["kind"], s.case["step"] == "train"
    a = [None if v is None else v.double().requires_grad_(train)
         for v in (s.x, s.y, s.w, s.b, s.gate, s.scale, s.w_next, s.b_next)]
    x, y, w, b, gate, scale, w_next, b_next = a
    branch = _norm64(y, w, b, kind)
    if gate is not None:
        branch = branch * gate
    if scale is not None:
        branch = branch * scale
    h = x + branch
    held = h + (h.detach().to(s.dtype).double() - h.detach())  # its gradient is h's
    n = _norm64(held, w_next, b_next, kind)
    if not train:
        return [h, n]
    grads = torch.autograd.grad([h, n], [v for v in a if v is not None],
                                [s.dh.double(), s.dn.double()])
    return [h.detach(), n.detach(), *grads]

"""Experts and linear layers in 8-bit integers, as measurable cases.

Weights are held as integers of -127..127 with a float32 scale for each output channel,
activations are brought to the same form row by row (a scale for each token) within the
calls, and products are sums of integers.  With s = max|v| / 127 (float32) of a row or
channel, v is held as s * q, q the integer nearest to v / s, ties to even.

A case is one pass through one operator's public entry point:

* ``op="rows"``: ``int8_rows`` and ``int8_rows_decode``, token rows to 8 bits and back.
* ``op="weight"``: ``int8_weight`` and ``int8_weight_decode``, a layer's or its experts'
  weights to 8 bits (what loading a model does) and back.
* ``op="product"``: ``int8_grouped_gemm_fn``, tokens by the weights of their experts, or of
  one linear layer (E = 1, no offsets).
* ``op="ffn"``: ``int8_swiglu_ffn_fn`` / ``int8_gelu_ffn_fn``, the experts' whole feed-forward
  block; the hidden values are held in the activations' type before they go to 8 bits.
* ``op="few"``: ``moe_few_tokens`` on 8-bit weights, a whole MoE layer for the few tokens of a
  decode step.

``step``: ``"infer"`` (forward) or ``"train"`` (forward and the tokens' gradient, with the
weights frozen and the rounding of activations passed straight through).

With ``own`` false the same is computed by elementary torch operations in 32 bits, with
integers next to a border decided in 64.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
LEAST = 2.0 ** -126  # of a scale


def _rows(name, dtype, A, f):
    return dict(name=name, op="rows", dtype=dtype, A=A, f=f)


def _weight(name, dtype, E, K, N):
    return dict(name=name, op="weight", dtype=dtype, E=E, K=K, N=N)


def _product(name, step, dtype, E, A, K, N):
    return dict(name=name, op="product", step=step, dtype=dtype, E=E, A=A, K=K, N=N)


def _ffn(name, step, dtype, ffn, E, A, d, f):
    return dict(name=name, op="ffn", step=step, dtype=dtype, ffn=ffn, E=E, A=A, d=d, f=f)


def _few(name, dtype, ffn, T, d, f, E, k, router):
    return dict(name=name, op="few", dtype=dtype, ffn=ffn, T=T, d=d, f=f, E=E, k=k, router=router)


def listed():
    return [
        # The tokens of a decode step before a product: one short launch.
        _rows("rows_step", "bf16", 16, 4096),
        # The experts' hidden rows at an odd width.
        _rows("rows_odd", "fp16", 40 * 768 + 1, 1365),
        # Loading the up projections of a large-hidden layer's experts.
        _weight("weight_wide", "bf16", 8, 4096, 14336),
        # Loading full-precision experts of unrounded 8 d / 3 widths.
        _weight("weight_odd", "fp32", 16, 512, 1365),
        # One token through one linear layer of the large-hidden model: latency.
        _product("product_one", "infer", "bf16", 1, 1, 4096, 14336),
        # Few, uneven experts in full precision, fine-tuned around frozen weights.
        _product("product_odd", "train", "fp32", 7, 5003, 300, 1365),
        # The down projections of a long prompt's tokens.
        _product("product_wide", "infer", "bf16", 8, 32768, 14336, 4096),
        # The repository's training shape in a forward pass: top-2 of 40 x 768 tokens.
        _ffn("ffn_base", "infer", "bf16", "swiglu", 8, 2 * 40 * 768, 512, 2048),
        # Fine-tuning around many narrow frozen experts.
        _ffn("ffn_fine", "train", "fp16", "gelu", 128, 8 * 1789, 2048, 768),
        # A long prompt through a large-hidden layer: the matrix products are all that counts.
        _ffn("ffn_wide", "infer", "bf16", "swiglu", 8, 32768, 4096, 14336),
        # One sequence decoding through the small configuration's layer: latency.
        _few("few_one", "bf16", "swiglu", 1, 512, 2048, 16, 2, True),
        # A full batch of decoding sequences through a large-hidden layer.
        _few("few_full", "bf16", "swiglu", 64, 4096, 14336, 8, 2, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case of the listed ones' ranges; rows and widths are any number."""
    kind = rng.choice(["rows", "weight", "product_few", "product", "product", "ffn_small",
                       "ffn_small", "ffn_fine", "ffn_wide", "few_small", "few_fine", "few_wide"])
    half = rng.choice(["bf16", "fp16"])
    any_type = rng.choice(["bf16", "fp16", "fp32"])
    ffn = rng.choice(["swiglu", "gelu"])
    step = rng.choice(["infer", "infer", "train"])
    d = rng.choice([128, 256, 300, 512, 1024])
    f = rng.choice([8 * d // 3, 4 * d])
    if kind == "rows":
        f = rng.choice([rng.randint(64, 2999), 512, 4096, 14336])
        c = _rows("", any_type, _log_int(rng, 1, 2 ** 27 // f), f)
    elif kind == "weight":
        K, N = rng.choice([(d, f), (f, d), (2048, 768), (4096, 14336)])
        c = _weight("", any_type, _log_int(rng, 1, min(64, 2 ** 28 // (K * N))), K, N)
    elif kind == "product_few":
        K, N = rng.choice([(d, f), (4096, 4096), (14336, 4096), (4096, 14336)])
        E = rng.choice([1, 1, 8])
        c = _product("", "infer", any_type, E, _log_int(rng, 1, 64 * E), K, N)
    elif kind == "product":
        K, N = rng.choice([(d, f), (f, d), (2048, 768), (4096, 4096), (4096, 14336)])
        E = rng.choice([1, 3, 8, 16])
        c = _product("", step, any_type, E, _log_int(rng, 256, min(65536, 2 ** 38 // (K * N))),
                     K, N)
    elif kind == "ffn_small":
        c = _ffn("", step, half, ffn, rng.choice([1, 4, 8, 16]), _log_int(rng, 64, 61440), d, f)
    elif kind == "ffn_fine":
        c = _ffn("", step, half, ffn, rng.choice([64, 128]), _log_int(rng, 256, 16384), 2048, 768)
    elif kind == "ffn_wide":
        c = _ffn("", step, half, ffn, 8, _log_int(rng, 256, 8192), 4096, 14336)
    elif kind == "few_small":
        c = _few("", half, ffn, _log_int(rng, 1, 64), d, f, rng.choice([4, 8, 16, 32]),
                 rng.choice([1, 2, 4]), rng.random() < 0.5)
    elif kind == "few_fine":
        c = _few("", half, ffn, _log_int(rng, 1, 64), 2048, 768, rng.choice([64, 128]), 8,
                 rng.random() < 0.5)
    else:
        c = _few("", half, ffn, _log_int(rng, 1, 60), 4096, 14336, 8, 2, True)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs


def _held(v, dim):
    """(integers, scales) of v along `dim`, as every operator here holds them."""
    v = v.float()
    most = v.abs().amax(dim, keepdim=True)
    s = (most / torch.full_like(most, 127.0)).clamp(min=LEAST)
    return torch.round(v.double() / s.double()).float(), s


def _blocks(q):
    """The integers of [E,K,N] in the order that the framework keeps: blocks of 64 columns by 64
    rows, [E, N / 64, K / 64, 4, 4, 16, 16], padded with zeros to 64 columns and 128 rows."""
    E, K, N = q.shape
    q = torch.nn.functional.pad(q, (0, -N % 64, 0, -K % 128))
    E, K, N = q.shape
    # k = 64 kb + 16 g + b, n = 64 nb + 16 i + 4 t + j
    q = q.view(E, K // 64, 4, 16, N // 64, 4, 4, 4).permute(0, 4, 1, 6, 2, 5, 7, 3)
    return q.reshape(E, N // 64, K // 64, 4, 4, 16, 16)


def _counts(A, E, seed):
    """Rows of each of E experts: uneven, and some of many have none."""
    g = torch.Generator().manual_seed(seed)
    p = torch.exp(0.25 * torch.randn(E, generator=g))
    if E > 2:
        p[E // 2] = 0.0
    owner = torch.multinomial(p, A, replacement=True, generator=g)
    return torch.bincount(owner, minlength=E)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, dt=dtype):
        return torch.empty(*shape, dtype=dt, device="cuda").normal_(0.0, std, generator=g)

    def weight(E, K, N):
        # trained weights' scale: activations of unit order; what a program keeps of them
        q, scale = _held(randn(E, K, N, std=K ** -0.5, dt=torch.float32), 1)
        q = q.to(torch.int8)
        return SimpleNamespace(q=q, scale=scale.view(E, N), blocks=_blocks(q), shape=(E, K, N))

    s = SimpleNamespace(case=case, dtype=dtype)
    op = case["op"]
    if op == "rows":
        s.x = randn(case["A"], case["f"])
        return s
    if op == "weight":
        s.W = randn(case["E"], case["K"], case["N"], std=case["K"] ** -0.5)
        return s
    if op == "few":
        T, d, f, E = (case[n] for n in ("T", "d", "f", "E"))
        s.x = randn(T, d)
        s.router = randn(E, d, std=d ** -0.5, dt=torch.float32) if case["router"] else None
        s.logits = None if case["router"] else randn(T, E, dt=torch.float32)
        s.weights = [weight(E, d, f) for _ in range(2 if case["ffn"] == "swiglu" else 1)]
        s.weights.append(weight(E, f, d))
        return s
    E, A = case["E"], case["A"]
    s.offsets = s.at = None
    if E > 1:
        n = _counts(A, E, seed)
        ends = n.cumsum(0)
        s.offsets = torch.cat([n.new_zeros(1), ends]).to(torch.int32).cuda()
        # the plain form's plan: every expert's rows, filled up to the longest one's, and back
        owner = torch.repeat_interleave(torch.arange(E), n)
        place = torch.arange(A) - (ends - n)[owner]
        rows = ((ends - n)[:, None] + torch.arange(int(n.max()))).clamp(max=A - 1)
        s.at = (rows.cuda(), owner.cuda(), place.cuda())
    if op == "product":
        s.x = randn(A, case["K"])
        s.weights = [weight(E, case["K"], case["N"])]
        outs = case["N"]
    else:
        d, f = case["d"], case["f"]
        s.x = randn(A, d)
        s.weights = [weight(E, d, f) for _ in range(2 if case["ffn"] == "swiglu" else 1)]
        s.weights.append(weight(E, f, d))
        outs = d
    if case["step"] == "train":
        s.dout = randn(A, outs)
    return s


# --------------------------------------------------------------------- run


def run(s):
    op = s.case["op"]
    if op == "rows":
        return _run_rows(s)
    if op == "weight":
        return _run_weight(s)
    if op == "few":
        return _run_few(s)
    return _run_grouped(s)


def _run_rows(s):
    if own:
        from nanotitan_amd.moe_ops import int8_rows, int8_rows_decode

        codes, scales = int8_rows(s.x)
        return [int8_rows_decode(codes, scales, s.x.shape[1], s.dtype), scales]
    q, scale = _held(s.x, 1)
    return [(q * scale).to(s.dtype), scale.view(-1)]


def _run_weight(s):
    if own:
        from nanotitan_amd.moe_ops import int8_weight, int8_weight_decode

        w = int8_weight(s.W)
        return [int8_weight_decode(w, s.dtype), w.scale]
    q, scale = _held(s.W, 1)
    return [(q * scale).to(s.dtype), scale.view(scale.shape[0], -1)]


def _handles(s):
    """The weights as the framework takes them."""
    from nanotitan_amd.moe_ops import Int8Weight

    return [Int8Weight(w.blocks, w.scale, w.shape) for w in s.weights]


def _run_grouped(s):
    train = s.case["step"] == "train"
    if own:
        from nanotitan_amd.moe_ops import (
            int8_gelu_ffn_fn,
            int8_grouped_gemm_fn,
            int8_swiglu_ffn_fn,
        )

        x = s.x.detach().requires_grad_(train)
        call = (int8_grouped_gemm_fn if s.case["op"] == "product" else
                int8_swiglu_ffn_fn if s.case["ffn"] == "swiglu" else int8_gelu_ffn_fn)
        out = call(x, *_handles(s), s.offsets)
        return [out, *torch.autograd.grad(out, x, s.dout)] if train else [out]
    if s.case["op"] == "product":
        outs = [_times(s, s.x, s.weights[0])]
        if train:
            outs.append(_times_t(s, s.dout.float(), s.weights[0]))
        return [o.to(s.dtype) for o in outs]
    h = _times(s, s.x, s.weights[0])
    if s.case["ffn"] == "swiglu":
        v = _times(s, s.x, s.weights[1])
        sg = 1.0 / (1.0 + torch.exp(-h))
        act = h * sg * v
    else:
        cdf = 0.5 * (1.0 + torch.erf(h * 0.5 ** 0.5))
        act = h * cdf
    act = act.to(s.dtype)  # as the hidden values are held
    outs = [_times(s, act, s.weights[-1])]
    if train:
        da = _times_t(s, s.dout.float(), s.weights[-1])
        if s.case["ffn"] == "swiglu":
            dx = (_times_t(s, da * v * sg * (1.0 + h * (1.0 - sg)), s.weights[0])
                  + _times_t(s, da * h * sg, s.weights[1]))
        else:
            slope = cdf + h * torch.exp(-0.5 * h * h) / math.sqrt(2.0 * math.pi)
            dx = _times_t(s, da * slope, s.weights[0])
        outs.append(dx)
    return [o.to(s.dtype) for o in outs]


def _by_expert(s, x, w):
    """x's rows times the matrix of each row's expert, in 32 bits."""
    if s.at is None:
        return x @ w[0]
    rows, owner, place = s.at
    return torch.matmul(x[rows], w)[owner, place]


def _times(s, x, w):
    q, scale = _held(x, 1)
    out = _by_expert(s, q, w.q.float())
    return out * scale * (w.scale if s.at is None else w.scale[s.at[1]])


def _times_t(s, dout, w):
    return _by_expert(s, dout, (w.q.float() * w.scale.unsqueeze(1)).transpose(1, 2).contiguous())


def _run_few(s):
    k = s.case["k"]
    if own:
        from nanotitan_amd.moe_ops import moe_few_tokens

        with torch.no_grad():
            out, gates, ids = moe_few_tokens(s.x, _handles(s), k, router_weight=s.router,
                                             logits=s.logits)
        return [out, gates, ids]
    logits = s.logits if s.router is None else s.x.float() @ s.router.t()
    # stable: equal logits go to the lower expert
    ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :k]
    top = logits.gather(1, ids)
    p = torch.exp(top - top[:, :1])
    gates = p / p.sum(-1, keepdim=True)
    # every expert on every token, weighted by a gate that is zero where it was not chosen
    dense = torch.zeros_like(logits).scatter_(1, ids, gates)
    qx, sx = _held(s.x, 1)
    up = [torch.matmul(qx, w.q.float()) * sx * w.scale.unsqueeze(1) for w in s.weights[:-1]]
    if s.case["ffn"] == "swiglu":
        h = up[0] / (1.0 + torch.exp(-up[0])) * up[1]  # [E,T,f]
    else:
        h = 0.5 * up[0] * (1.0 + torch.erf(up[0] * 0.5 ** 0.5))
    qh, sh = _held(h.to(s.dtype), 2)  # as the hidden values are held
    w = s.weights[-1]
    y = torch.matmul(qh, w.q.float()) * sh * w.scale.unsqueeze(1)
    out = (dense.t().unsqueeze(-1) * y).sum(0)
    return [out.to(s.dtype), gates, ids.to(torch.int32)]


# -------------------------------------------------------------------- work


def work(case):
    c = case
    b = torch.finfo(DTYPES[c["dtype"]]).bits // 8
    if c["op"] in ("rows", "weight"):
        # to 8 bits and back: values in and out, the integers written and read
        n = c["A"] * c["f"] if c["op"] == "rows" else c["E"] * c["K"] * c["N"]
        scales = c["A"] if c["op"] == "rows" else c["E"] * c["N"]
        return {"bytes": n * (2 * b + 2) + 8 * scales, "flops": 6 * n}
    if c["op"] == "few":
        T, d, f, E, k = (c[n] for n in ("T", "d", "f", "E", "k"))
        mats = 3 if c["ffn"] == "swiglu" else 2
        # the chosen experts' weights, expected under uniform routing
        live = E * (1.0 - (1.0 - k / E) ** T)
        router = E * d * 4 if c["router"] else T * E * 4
        scales = 4 * ((mats - 1) * f + d)
        return {"bytes": int((mats * d * f + scales) * live + 2 * T * d * b + router + 8 * T * k),
                "flops": 2 * mats * T * k * d * f}
    train = 2 if c["step"] == "train" else 1
    E, A = c["E"], c["A"]
    live = min(E - (E > 2), A)
    if c["op"] == "product":
        K, N = c["K"], c["N"]
        weights, flops = K * N + 4 * N, 2 * K * N
        ins = outs = (K + N) * b
    else:
        d, f = c["d"], c["f"]
        mats = 3 if c["ffn"] == "swiglu" else 2
        weights, flops = mats * d * f + 4 * ((mats - 1) * f + d), 2 * mats * d * f
        ins = outs = 2 * d * b
    return {"bytes": live * weights + A * (ins + (outs if train == 2 else 0)),
            "flops": train * A * flops}


# ------------------------------------------------------------------- exact


def _held64(v, dim):
    """What 8 bits hold of v: float32 scales, every value the nearest multiple of its own."""
    v = v.double()
    most = v.abs().amax(dim, keepdim=True)
    s = (most / torch.full_like(most, 127.0)).float().clamp(min=LEAST).double()
    return torch.round(v / s) * s, s


def _matrices(w, e):
    return [m.q[e].double() * m.scale[e].double() for m in w]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rows":
        held, scale = _held64(s.x, 1)
        return [held, scale.view(-1)]
    if case["op"] == "weight":
        parts = [_held64(w, 0) for w in s.W]
        return [torch.stack([h for h, _ in parts]), torch.stack([c.view(-1) for _, c in parts])]
    if case["op"] == "few":
        return _exact_few(s)
    train = case["step"] == "train"
    if s.offsets is None:
        ends = [0, case["A"]]
    else:
        ends = s.offsets.tolist()
    outs, grads = [], []
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        if a == b:
            continue
        m = _matrices(s.weights, e)
        dout = s.dout[a:b].double() if train else None
        if case["op"] == "product":
            outs.append(_held64(s.x[a:b], 1)[0] @ m[0])
            if train:
                grads.append(dout @ m[0].t())
            continue
        y, back = _block64(s.x[a:b], m, s.dtype)
        outs.append(y)
        if train:
            grads.append(back(dout))
    return [torch.cat(outs), torch.cat(grads)] if train else [torch.cat(outs)]


def _block64(x, m, dtype):
    """An expert's feed-forward block on rows x, and its gradient to them."""
    pre = [(_held64(x, 1)[0] @ w).requires_grad_() for w in m[:-1]]
    if len(pre) == 2:
        act = torch.nn.functional.silu(pre[0]) * pre[1]
    else:
        act = torch.nn.functional.gelu(pre[0])
    y = _held64(act.detach().to(dtype), 1)[0] @ m[-1]

    def back(dout):
        d = torch.autograd.grad(act, pre, dout @ m[-1].t())
        return sum(g @ w.t() for g, w in zip(d, m))

    return y, back


def _exact_few(s):
    x = s.x.double()
    logits = s.logits.double() if s.router is None else x @ s.router.double().t()
    ids = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :s.case["k"]]
    gates = logits.gather(1, ids).softmax(-1)
    out = torch.zeros_like(x)
    for e in torch.unique(ids).tolist():
        t, j = torch.nonzero(ids == e, as_tuple=True)
        y, _ = _block64(s.x[t], _matrices(s.weights, e), s.dtype)
        out.index_add_(0, t, gates[t, j].unsqueeze(1) * y)
    return [out, gates, ids.to(torch.int32)]

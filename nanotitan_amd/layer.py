"""MoE layer on the HIP expert path: the drop-in for the reference's CUDA backend.

* ``HIPMoEBackend(cfg, experts, router, spec)`` — the dataflow of the
  reference's ``CUDAMoEBackend.forward`` (src/model/cuda_backend.py:17-81):
  router in ``cfg.moe_router_dtype``, fp32 softmax / top-k / renorm, count,
  offsets, pack, experts, combine, cast, and ``MoELayerStats``. It takes the
  four-argument constructor that ``MoE.__init__`` uses
  (src/model/feed_fwd.py:142; the reference class only accepts three).
  The router kernel emits the per-block expert counts, offsets + pack run as
  one native call after it, and the combine writes
  the activation dtype directly (same values as combine-to-fp32-then-cast).
* ``ExpertFFN(cfg, spec)`` — SwiGLU experts with ``[E,d,f]`` / ``[E,f,d]``
  weights (src/model/feed_fwd.py:39-122), three grouped GEMMs.
* ``GeluExpertFFN(cfg, spec)`` — the 2-GEMM up -> GELU -> down FFN the
  benchmark configs specify, with the activation fused into the GEMMs.
* ``Int8ExpertFFN(experts)`` — either of them on frozen 8-bit integer weights.
* ``MoE(cfg, spec)`` — router + experts + backend (src/model/feed_fwd.py:128-152);
  ``MoE.decode`` runs the layer on the few tokens of a decode step, and
  ``MoE.quantize_experts`` puts its experts on 8-bit weights.
* ``MoEBlock(cfg, spec)`` — the MoE half of a transformer layer: norm, MoE, norm,
  gate, residual scale and sum (src/model/model.py:205-211).
* ``route(logits, top_k)`` — fp32 softmax, top-k with ties to the lower
  expert id, renormalised gates, int32 ids.

``cfg.ffn_checkpoint8 = True`` has the experts keep their activations in 8
bits for the backward.

Only the HIP path exists here; any other ``moe_backend`` raises.
"""

from __future__ import annotations

from dataclasses import dataclass, field

import torch
import torch.nn as nn
from torch.profiler import record_function

from nanotitan_amd.capi import NT_FEW_TOKENS_MAX
from nanotitan_amd.moe_ops import (
    combine_inv_fn,
    grouped_gelu_ffn8_fn,
    grouped_gelu_ffn_fn,
    int8_gelu_ffn_fn,
    int8_swiglu_ffn_fn,
    int8_weight,
    Int8Weight,
    moe_few_tokens,
    post_norm_fn,
    pre_norm_fn,
    route_dispatch_fn,
    route_fn,
    router_aux_fn,
    router_gate_fn,
    router_stats_fn,
    swiglu_ffn8_fn,
    swiglu_ffn_fn,
)

HIP_BACKENDS = ("hip", "cuda")  # "cuda" is accepted so reference configs select this path


@dataclass
class ModelShardSpec:
    """Expert range of this rank (reference src/model/utils.py:10-20); ep_size is 1 here."""

    layer_start: int = 0
    layer_end: int = 1
    has_token_embed: bool = False
    has_pos_embed: bool = False
    has_unembed_head: bool = False
    per_rank_expert: int = 1
    start_expert_id: int = 0
    end_expert_id: int = 1
    ep_size: int = 1
    ep_group: object | None = None


@dataclass
class MoELayerStats:
    """Routing statistics and the load-balancing loss (reference src/model/utils.py:70-93)."""

    tokens_per_expert: torch.Tensor
    probs_per_expert: torch.Tensor
    cfg: object
    aux_loss: torch.Tensor | None = field(default=None)

    def __post_init__(self):
        self.num_tokens = self.probs_per_expert.shape[0]
        self.total_assignments = self.tokens_per_expert.sum()
        self.ass_frac_per_expert = self.tokens_per_expert.float() / self.total_assignments
        self.probs_per_expert = self.probs_per_expert.mean(dim=0)
        self.aux_loss = (
            self.cfg.router_alpha
            * self.cfg.num_experts
            * torch.sum(self.ass_frac_per_expert * self.probs_per_expert)
        )

    @classmethod
    def from_logits(cls, tokens_per_expert, logits, cfg, router=None):
        """The same statistics from the float32 router logits, in one kernel.

        ``router``: (float32 tokens, weight) where the gradient goes to the weight of
        the linear that gives these logits; else it goes to ``logits``.
        """
        stats = cls.__new__(cls)
        stats.tokens_per_expert = tokens_per_expert
        stats.cfg = cfg
        stats.num_tokens = logits.shape[0]
        coef = cfg.router_alpha * cfg.num_experts
        (stats.total_assignments, stats.ass_frac_per_expert, stats.probs_per_expert,
         stats.aux_loss) = (router_stats_fn(logits, tokens_per_expert, coef) if router is None
                            else router_aux_fn(logits, *router, tokens_per_expert, coef))
        return stats


def route(logits: torch.Tensor, top_k: int):
    """(gates f32 [T,k], ids int32 [T,k]) from the fused router kernel.

    Reference src/model/cuda_backend.py:30-37: fp32 softmax, torch.topk,
    renormalise. The kernel selects the k largest logits (the same set as the
    k largest probabilities; ties go to the lower expert id, where torch.topk
    leaves the order unspecified) and returns the selected probabilities
    renormalised to sum 1.
    """
    return route_fn(logits.float().contiguous(), top_k)


def _check_backend(cfg):
    backend = getattr(cfg, "moe_backend", "hip")
    if backend not in HIP_BACKENDS:
        raise ValueError(f"moe_backend={backend!r}: this package implements only the HIP path")


class ExpertFFN(nn.Module):
    """SwiGLU experts: silu(X W_gate) * (X W_val), then W_out (reference feed_fwd.py:39-122)."""

    def __init__(self, cfg, spec):
        super().__init__()
        _check_backend(cfg)
        self.cfg = cfg
        self.spec = spec
        E, d, f = spec.per_rank_expert, cfg.d_model, cfg.ffn_in
        self.W_gate = nn.Parameter(torch.empty(E, d, f, dtype=cfg.dtype))
        self.W_val = nn.Parameter(torch.empty(E, d, f, dtype=cfg.dtype))
        self.W_out = nn.Parameter(torch.empty(E, f, d, dtype=cfg.dtype))
        for p in (self.W_gate, self.W_val, self.W_out):
            nn.init.kaiming_normal_(p, mode="fan_in", nonlinearity="relu")

    def forward(self, packed_X, expert_offset):
        # Gate and value GEMMs in one kernel with silu(gate) * value in its
        # epilogue; the backward fuses the activation's gradient likewise.
        ffn = swiglu_ffn8_fn if getattr(self.cfg, "ffn_checkpoint8", False) else swiglu_ffn_fn
        return ffn(packed_X, self.W_gate, self.W_val, self.W_out, expert_offset)

    def parameter_count(self) -> int:
        return sum(p.numel() for p in self.parameters())


class GeluExpertFFN(nn.Module):
    """Up -> GELU (erf) -> down experts, the FFN of the benchmark configs."""

    def __init__(self, cfg, spec, std: float = 0.02):
        super().__init__()
        _check_backend(cfg)
        self.cfg = cfg
        self.spec = spec
        E, d, f = spec.per_rank_expert, cfg.d_model, cfg.ffn_in
        self.W_up = nn.Parameter(torch.randn(E, d, f).mul_(std).to(cfg.dtype))
        self.W_down = nn.Parameter(torch.randn(E, f, d).mul_(std).to(cfg.dtype))

    def forward(self, packed_X, expert_offset):
        ffn = (grouped_gelu_ffn8_fn if getattr(self.cfg, "ffn_checkpoint8", False)
               else grouped_gelu_ffn_fn)
        return ffn(packed_X, self.W_up, self.W_down, expert_offset)


class Int8ExpertFFN(nn.Module):
    """An ``ExpertFFN``'s or ``GeluExpertFFN``'s weights, frozen, in 8-bit integers.

    Tokens and hidden values go to 8 bits row by row; the tokens get their gradient, the weights
    none. The weights are buffers: two a projection, ``<name>_codes`` and ``<name>_scale``, the
    float32 scales as the int32 of their bits, which a cast of the module to another float type
    leaves alone. ``cfg.ffn_checkpoint8`` does not apply: what the backward keeps is gate and
    value, or gelu', in float32. ``cfg.int8_exact_gradient = False`` rounds the weights to 16
    bits in a 16-bit gradient, which is faster (``int8_swiglu_ffn_fn``).
    """

    def __init__(self, experts):
        super().__init__()
        if type(experts) is ExpertFFN:
            self.names = ("W_gate", "W_val", "W_out")
        elif type(experts) is GeluExpertFFN:
            self.names = ("W_up", "W_down")
        else:
            raise RuntimeError(f"8-bit weights of this package's experts, not "
                               f"{type(experts).__name__}")
        self.cfg, self.spec = experts.cfg, experts.spec
        self.shapes = {}
        for name in self.names:
            w = int8_weight(getattr(experts, name))
            self.shapes[name] = w.shape
            self.register_buffer(f"{name}_codes", w.codes)
            self.register_buffer(f"{name}_scale", w.scale.view(torch.int32))
        self.train(experts.training)

    def weights(self):
        """The projections' Int8Weights, as ``moe_few_tokens`` and the ``int8_*_ffn_fn`` take them."""
        return tuple(Int8Weight(getattr(self, f"{name}_codes"),
                                getattr(self, f"{name}_scale").view(torch.float32),
                                self.shapes[name]) for name in self.names)

    def forward(self, packed_X, expert_offset):
        ffn = int8_swiglu_ffn_fn if len(self.names) == 3 else int8_gelu_ffn_fn
        return ffn(packed_X, *self.weights(), expert_offset,
                   getattr(self.cfg, "int8_exact_gradient", True))


def moe_forward_from_logits(x_flat, logits, experts, num_experts, top_k):
    """Hot path from router logits: route, dispatch, experts, combine (output in x's dtype).

    Returns (out [T,d], counts [E], gates [T,k]).
    """
    # The router kernel also counts the tokens per expert and per dispatch
    # block, so the dispatch starts at its scan; in the backward, the pack
    # backward also writes the router's gradient.
    with record_function("moe/topK_pack_tokens"):
        gates, idx, packed_X, packed_w, counts, offsets, _token_id, inv = route_dispatch_fn(
            logits.float().contiguous(), top_k, x_flat, num_experts
        )
    with record_function("moe/expert_compute"):
        y = experts(packed_X, offsets)
    with record_function("moe/combine_tokens"):
        out = combine_inv_fn(y, inv, packed_w, x_flat.dtype)
    return out, counts, gates


def _plain_router(router, flat) -> bool:
    """Whether calling ``router`` is exactly float32 ``flat @ weight.T``, with no
    hook, subclass, cast or bias that a second call could make differ."""
    hooks = (router._forward_hooks, router._forward_pre_hooks, router._backward_hooks,
             router._backward_pre_hooks)
    return (type(router) is nn.Linear and router.bias is None and not any(hooks)
            and "forward" not in router.__dict__
            and not nn.modules.module._has_any_global_hook()
            and type(router.weight) is nn.Parameter and router.weight.dtype == torch.float32
            and type(flat) is torch.Tensor and flat.is_cuda and router.weight.is_cuda
            and flat.dtype in (torch.float32, torch.float16, torch.bfloat16)
            and flat.shape[0] > 0 and not torch.is_autocast_enabled())


def _plain_experts(experts) -> bool:
    """Whether calling ``experts`` without gradients is its class's ``forward`` and nothing else."""
    return (not experts._forward_hooks and not experts._forward_pre_hooks
            and "forward" not in experts.__dict__
            and not nn.modules.module._has_any_global_hook())


def _hung_on(module) -> bool:
    """Whether hooks hang on a module, or a forward stands in place of its class's."""
    return any((module._forward_hooks, module._forward_pre_hooks, module._backward_hooks,
                module._backward_pre_hooks)) or "forward" in module.__dict__


class HIPMoEBackend:
    """Reference CUDAMoEBackend dataflow (src/model/cuda_backend.py:11-81) on the HIP path."""

    def __init__(self, cfg, experts: nn.Module, router: nn.Linear, spec=None):
        _check_backend(cfg)
        self.cfg = cfg
        self.router = router
        self.experts = experts
        self.spec = spec

    def forward(self, x: torch.Tensor):
        batch, seq_len, d_model = x.shape
        flat = x.reshape(-1, d_model)
        router_dtype = self.router.weight.dtype
        plain = (_plain_router(self.router, flat)
                 and type(self.cfg.router_alpha * self.cfg.num_experts) in (int, float))
        with record_function("moe/router"):
            # Aux-loss logits come from a second router pass on detached tokens
            # (src/model/cuda_backend.py:40-41), so the aux grad reaches only
            # the router. A plain linear router computes the same logits both
            # times: the second pass is then only its gradient (RouterAuxFN),
            # and nothing at all without gradients.
            grad = torch.is_grad_enabled()
            one_pass = plain and (not grad or self.router.weight.shape[0] <= 32)
            if one_pass and grad:
                flat32 = flat.to(router_dtype)
                logits = router_gate_fn(flat, flat32, self.router.weight)
            else:
                logits = self.router(flat.to(router_dtype))
        if one_pass:
            aux_logits = logits
        else:
            aux_logits = self.router(flat.detach().to(router_dtype))
        out, counts, _ = moe_forward_from_logits(
            flat, logits, self.experts, self.cfg.num_experts, self.cfg.top_k
        )
        if plain:
            stats = MoELayerStats.from_logits(
                counts.detach(), aux_logits, self.cfg,
                router=(flat32, self.router.weight) if one_pass and grad else None)
        else:
            stats = MoELayerStats(tokens_per_expert=counts.detach(),
                                  probs_per_expert=aux_logits.softmax(dim=-1), cfg=self.cfg)
        return out.reshape(batch, seq_len, d_model), stats


class MoE(nn.Module):
    """Router + experts + HIP backend (reference src/model/feed_fwd.py:128-152)."""

    def __init__(self, cfg, spec=None, ffn: str = "swiglu"):
        super().__init__()
        _check_backend(cfg)
        if spec is None:
            spec = ModelShardSpec(per_rank_expert=cfg.num_experts, end_expert_id=cfg.num_experts)
        self.cfg = cfg
        self.spec = spec
        self.experts = ExpertFFN(cfg, spec) if ffn == "swiglu" else GeluExpertFFN(cfg, spec)
        router_dtype = getattr(cfg, "moe_router_dtype", torch.float32)
        self.router = nn.Linear(cfg.d_model, cfg.num_experts, bias=False, dtype=router_dtype)
        self.moe_backend = HIPMoEBackend(cfg, self.experts, self.router, spec)

    def forward(self, x):
        return self.moe_backend.forward(x)

    @torch.no_grad()
    def quantize_experts(self):
        """Puts the experts' weights into 8-bit integers, in place (``Int8ExpertFFN``): the module
        then has no expert parameters, and an optimizer made before still holds the old ones.
        Hooks on the experts, or a forward put in place of theirs, would be lost: it raises then.
        Returns self."""
        if type(self.experts) is not Int8ExpertFFN:
            if _hung_on(self.experts):
                raise RuntimeError("quantize_experts replaces the experts: remove their hooks, or "
                                   "the forward put in place of theirs, and add them to the new "
                                   "ones")
            self.experts = Int8ExpertFFN(self.experts)
            self.moe_backend.experts = self.experts
        return self

    @torch.no_grad()
    def decode(self, x):
        """The layer's output for the few tokens (at most 64 in all) of a decode step.

        x [B,S,d] -> [B,S,d], the values of ``forward`` up to the roundings that the one
        kernel path does not make; no statistics, no gradients. Hooks on the router run, and
        hooks on the experts (or a forward put in place of theirs) too, by the full path;
        those on this module belong to ``forward``.
        """
        e = self.experts
        if type(e) is ExpertFFN:
            weights = (e.W_gate, e.W_val, e.W_out)
        elif type(e) is GeluExpertFFN:
            weights = (e.W_up, e.W_down)
        elif type(e) is Int8ExpertFFN:
            weights = e.weights()
        else:
            raise RuntimeError(f"decode runs this package's experts, not {type(e).__name__}")
        flat = x.reshape(-1, x.shape[-1]).contiguous()
        if flat.shape[0] > NT_FEW_TOKENS_MAX:  # whatever hangs on the parts
            raise RuntimeError(f"decode takes at most {NT_FEW_TOKENS_MAX} tokens, "
                               f"got {flat.shape[0]}")
        plain = _plain_experts(e)
        if plain and _plain_router(self.router, flat):
            route = {"router_weight": self.router.weight}
        else:
            logits = self.router(flat.to(self.router.weight.dtype))
            if not plain:
                return moe_forward_from_logits(flat, logits, e, self.cfg.num_experts,
                                               self.cfg.top_k)[0].view(x.shape)
            route = {"logits": logits.float().contiguous()}
        return moe_few_tokens(flat, weights, self.cfg.top_k, **route)[0].view(x.shape)


class MoEBlock(nn.Module):
    """The MoE half of a transformer layer, h = x + scale * gate * N(MoE(N(x))).

    The reference's layer is x + ffn(ffn_norm(x)) (src/model/model.py:205-211): ``norm``
    "layer", ``post_norm`` False. ``norm`` is "rms" or "layer"; ``post_norm`` adds the norm
    after the MoE; ``residual_scale`` a learned scale per channel of that initial value; a
    gate is an input of ``forward``. Parameters are of cfg.dtype.

    Blocks that follow each other share a pass: ``forward(x, following=block)`` also
    returns ``block``'s first norm of h, which goes to it as ``normed``.
    """

    def __init__(self, cfg, spec=None, ffn: str = "swiglu", norm: str = "rms",
                 post_norm: bool = True, residual_scale: float | None = None, eps: float = 1e-6):
        super().__init__()
        if norm not in ("rms", "layer"):
            raise ValueError(f"norm={norm!r}: expected 'rms' or 'layer'")
        self.moe = MoE(cfg, spec, ffn=ffn)
        self.norm, self.eps = norm, eps

        def param(on, value):
            return nn.Parameter(torch.full((cfg.d_model,), value, dtype=cfg.dtype)) if on else None

        layer = norm == "layer"
        self.pre_weight, self.pre_bias = param(True, 1.0), param(layer, 0.0)
        self.post_weight = param(post_norm, 1.0)
        self.post_bias = param(post_norm and layer, 0.0)
        self.scale = param(residual_scale is not None, residual_scale)

    def _run(self, moe, x, normed, gate, following):
        if following is not None and (following.norm, following.eps) != (self.norm, self.eps):
            raise ValueError("a following block's norm must be of this block's kind and eps")
        if normed is None:
            normed = pre_norm_fn(x, self.pre_weight, self.pre_bias, self.norm, self.eps,
                                 self.pre_weight.dtype)
        y, *stats = moe(normed)
        nxt = (None, None) if following is None else (following.pre_weight, following.pre_bias)
        h = post_norm_fn(x, y, self.post_weight, self.post_bias, gate=gate, scale=self.scale,
                         next_weight=nxt[0], next_bias=nxt[1], kind=self.norm, eps=self.eps)
        return (*(h if following is not None else (h, None)), *stats)

    def forward(self, x, normed=None, gate=None, following=None):
        """x [B,S,d] -> (h, the following block's normed h or None, MoELayerStats)."""
        return self._run(self.moe, x, normed, gate, following)

    @torch.no_grad()
    def decode(self, x, normed=None, gate=None, following=None):
        """The same for few tokens (``MoE.decode``): (h, the following block's normed h or None)."""
        return self._run(lambda n: (self.moe.decode(n),), x, normed, gate, following)

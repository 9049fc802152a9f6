"""Autograd surface of the MoE expert path.

Same function names, argument orders and gradient contracts as the
reference's ``src/model/moe_ops.py:10-125``:

* ``pack_tokens_fn(X, topk_weights, topk_experts, expert_offset_cpy)``
  -> (packed_X, packed_tokenId, packed_expert, packed_topk_weights);
  backward returns (X_grad, topk_weights_grad, None, None).
* ``combine_tokens_fn(packed_expert_outputs, packed_tokenId,
  packed_topk_weights, num_tokens, hidden_dim)`` -> float32 [T, d];
  backward casts the incoming grad to float32 contiguous and returns
  (expert_output_grad, None, packed_topk_weights_grad, None, None).
* ``grouped_gemm_fn(X, weight, expert_offset)`` applies
  ``GroupedGEMM_FN.apply(X, expert_offset, weight)``; backward returns
  (dX, None, dW).

Every op runs the HIP kernels through ``get_hip_extension()``; a missing
extension raises RuntimeError, never a silent fallback.

The layer uses additional Functions built on the inverse map the pack
writes: ``RouteCountFN`` (router gate that also counts the tokens per expert
and dispatch block), ``DispatchFN`` (count + offsets + pack, or offsets + pack
from RouteCountFN's counts) and ``CombineInvFN`` (combine whose backward reads
each token's grad row once). They compute the same values as pack_tokens_fn /
combine_tokens_fn on the same inputs.

Beside that path: ``moe_few_tokens`` (the whole layer for a decode step),
``pre_norm_fn`` / ``post_norm_fn`` (norms, gate and residual of a block) and
``checkpoint8`` / ``gelu8_fn`` / ``swiglu8_fn`` with the experts' FFNs on them
(activations kept in 8 bits). The norms' and 8-bit activations' Functions are
in the extension.

``int8_weight`` and the ``int8_*_fn`` run experts and linear layers on 8-bit
integer weights, with the tokens brought to 8 bits row by row.
"""

from __future__ import annotations

import functools
from typing import Any, NamedTuple

import torch

from nanotitan_amd.extension import get_hip_extension


def combine_tokens_fn(
    packed_expert_outputs, packed_tokenId, packed_topk_weights, num_tokens, hidden_dim
):
    return CombineTokensFN.apply(
        packed_expert_outputs, packed_tokenId, packed_topk_weights, num_tokens, hidden_dim
    )


def pack_tokens_fn(X, topk_weights, topk_experts, expert_offset_cpy):
    return PackTokensFN.apply(X, topk_weights, topk_experts, expert_offset_cpy)


def grouped_gemm_fn(X, weight, expert_offset):
    return GroupedGEMM_FN.apply(X, expert_offset, weight)


class PackTokensFN(torch.autograd.Function):
    """Reference: src/model/moe_ops.py:40-73."""

    @staticmethod
    def forward(ctx, X, topk_weights, topk_experts, expert_offset_cpy) -> tuple:
        ext = get_hip_extension()
        packed_X, packed_tokenId, packed_expert, packed_topk_weights = ext.pack_tokens_kernel(
            X, topk_weights, topk_experts, expert_offset_cpy
        )
        ctx.save_for_backward(packed_tokenId, packed_expert, topk_experts)
        ctx.mark_non_differentiable(packed_tokenId, packed_expert)
        return packed_X, packed_tokenId, packed_expert, packed_topk_weights

    @staticmethod
    def backward(ctx, packed_X_grad, packed_tokenId_grad, packed_expert_grad,
                 packed_topk_weights_grad) -> Any:
        ext = get_hip_extension()
        packed_tokenId, packed_expert, topk_experts = ctx.saved_tensors
        if packed_topk_weights_grad is None:
            packed_topk_weights_grad = torch.zeros(
                packed_tokenId.shape, dtype=torch.float32, device=packed_tokenId.device
            )
        if packed_X_grad is None:
            raise RuntimeError("pack_tokens_fn backward needs a gradient for packed_X")
        X_grad, topk_weights_grad = ext.pack_kernel_backward(
            packed_X_grad.contiguous(),
            packed_topk_weights_grad.contiguous(),
            packed_tokenId,
            packed_expert,
            topk_experts,
        )
        return X_grad, topk_weights_grad, None, None


class CombineTokensFN(torch.autograd.Function):
    """Reference: src/model/moe_ops.py:76-104."""

    @staticmethod
    def forward(ctx, packed_expert_outputs, packed_tokenId, packed_topk_weights, num_tokens,
                hidden_dim) -> torch.Tensor:
        ext = get_hip_extension()
        pool = ext.combine_tokens_kernel(
            packed_expert_outputs, packed_tokenId, packed_topk_weights, num_tokens, hidden_dim
        )
        ctx.save_for_backward(packed_expert_outputs, packed_tokenId, packed_topk_weights)
        ctx.hidden_dim = hidden_dim
        return pool

    @staticmethod
    def backward(ctx, d_resid_stream) -> tuple:
        ext = get_hip_extension()
        packed_expert_outputs, packed_tokenId, packed_topk_weights = ctx.saved_tensors
        expert_output_grad, packed_topk_weights_grad = ext.combine_kernel_backward(
            packed_expert_outputs,
            packed_tokenId,
            packed_topk_weights,
            d_resid_stream.to(torch.float32).contiguous(),
            ctx.hidden_dim,
        )
        return expert_output_grad, None, packed_topk_weights_grad, None, None


class GroupedGEMM_FN(torch.autograd.Function):
    """Reference: src/model/moe_ops.py:107-125."""

    @staticmethod
    def forward(ctx, X, expert_offset, weight) -> torch.Tensor:
        ext = get_hip_extension()
        ctx.save_for_backward(X, expert_offset, weight)
        return ext.grouped_gemm_kernel(X, expert_offset, weight)

    @staticmethod
    def backward(ctx, out_grad) -> tuple:
        ext = get_hip_extension()
        X, expert_offset, weight = ctx.saved_tensors
        out_grad = out_grad.contiguous()
        dX = dW = None
        if ctx.needs_input_grad[0] and ctx.needs_input_grad[2]:
            # one call: the dW may run beside the dX (same values as the two calls)
            dW, dX = ext.bwd_grouped_gemm_dW_dX(X, weight, expert_offset, out_grad)
        elif ctx.needs_input_grad[0]:
            dX = ext.bwd_grouped_gemm_dX_kernel(weight, expert_offset, out_grad)
        elif ctx.needs_input_grad[2]:
            dW = ext.bwd_grouped_gemm_dW_kernel(X, expert_offset, out_grad)
        return dX, None, dW


class GroupedGeluFFN_FN(torch.autograd.Function):
    """Expert FFN up -> GELU (erf) -> down on the grouped GEMM, activation fused.

    Forward: (a, g) = grouped_gemm_gelu(X, W_up) — a = gelu(h) and
    g = gelu'(h) for h = X W_up, from one kernel — then y = a W_down.
    Backward: dH = (dy W_down^T) * g from one kernel, then the three
    remaining grouped GEMMs. The values of grouped_gemm_fn +
    torch.nn.functional.gelu + grouped_gemm_fn (the reference's ExpertFFN
    dataflow, src/model/feed_fwd.py:102-112, with the configs' GELU), except
    that gelu'(h) is rounded to the activation dtype before the multiply;
    backward returns (dX, None, dW_up, dW_down).
    """

    @staticmethod
    def forward(ctx, X, expert_offset, W_up, W_down):
        ext = get_hip_extension()
        a, g = ext.grouped_gemm_gelu(X, expert_offset, W_up)
        y = ext.grouped_gemm_kernel(a, expert_offset, W_down)
        ctx.save_for_backward(X, expert_offset, W_up, W_down, a, g)
        return y

    @staticmethod
    def backward(ctx, dy):
        ext = get_hip_extension()
        X, expert_offset, W_up, W_down, a, g = ctx.saved_tensors
        dy = dy.contiguous()
        dX = dW_up = dW_down = None
        need_dH = ctx.needs_input_grad[0] or ctx.needs_input_grad[2]
        # Each projection's dW and dX in one call: a dW with few 256x256
        # tiles runs beside its dX in one kernel launch (same values).
        if ctx.needs_input_grad[3] and need_dH:
            dW_down, dH = ext.bwd_grouped_gemm_dW_dX_gelu(a, W_down, expert_offset, dy, g)
        elif ctx.needs_input_grad[3]:
            dW_down = ext.bwd_grouped_gemm_dW_kernel(a, expert_offset, dy)
        elif need_dH:
            dH = ext.bwd_grouped_gemm_dX_gelu(W_down, expert_offset, dy, g)
        if ctx.needs_input_grad[0] and ctx.needs_input_grad[2]:
            dW_up, dX = ext.bwd_grouped_gemm_dW_dX(X, W_up, expert_offset, dH)
        elif ctx.needs_input_grad[0]:
            dX = ext.bwd_grouped_gemm_dX_kernel(W_up, expert_offset, dH)
        elif ctx.needs_input_grad[2]:
            dW_up = ext.bwd_grouped_gemm_dW_kernel(X, expert_offset, dH)
        return dX, None, dW_up, dW_down


def grouped_gelu_ffn_fn(X, W_up, W_down, expert_offset):
    return GroupedGeluFFN_FN.apply(X, expert_offset, W_up, W_down)


class SwiGLUFFN_FN(torch.autograd.Function):
    """The reference's SwiGLU ExpertFFN on fused grouped GEMMs.

    Forward: (h, g, v) = grouped_gemm_swiglu(X, W_gate, W_val) — the gate and
    value GEMMs in one kernel whose epilogue writes gate, value and
    hidden = silu(gate) * value — then y = h W_out. Backward:
    (dgate, dvalue) from one kernel (dhidden = dy W_out^T and the SwiGLU
    backward in its epilogue), dX = dgate W_gate^T + dvalue W_val^T as one
    GEMM over the concatenated reduction, and the three weight gradients.
    The values of the reference's _forward_cuda (src/model/feed_fwd.py:102-112:
    grouped_gemm_fn, grouped_gemm_fn, silu(gate) * value, grouped_gemm_fn),
    rounded where it rounds, except that the two dX products are summed
    before the one rounding; backward returns
    (dX, None, dW_gate, dW_val, dW_out).
    """

    @staticmethod
    def forward(ctx, X, expert_offset, W_gate, W_val, W_out):
        ext = get_hip_extension()
        h, g, v = ext.grouped_gemm_swiglu(X, expert_offset, W_gate, W_val)
        y = ext.grouped_gemm_kernel(h, expert_offset, W_out)
        ctx.save_for_backward(X, expert_offset, W_gate, W_val, W_out, h, g, v)
        return y

    @staticmethod
    def backward(ctx, dy):
        ext = get_hip_extension()
        X, expert_offset, W_gate, W_val, W_out, h, g, v = ctx.saved_tensors
        dy = dy.contiguous()
        dX = dW_gate = dW_val = dW_out = None
        need_d = any(ctx.needs_input_grad[i] for i in (0, 2, 3))
        # Paired calls (a dW with few tiles runs beside its dX in one launch).
        if ctx.needs_input_grad[4] and need_d:
            dW_out, dg, dv = ext.bwd_grouped_gemm_dW_dX_swiglu(h, W_out, expert_offset, dy, g, v)
        elif ctx.needs_input_grad[4]:
            dW_out = ext.bwd_grouped_gemm_dW_kernel(h, expert_offset, dy)
        elif need_d:
            dg, dv = ext.bwd_grouped_gemm_dX_swiglu(W_out, expert_offset, dy, g, v)
        if ctx.needs_input_grad[0] and ctx.needs_input_grad[2]:
            dW_gate, dX = ext.bwd_grouped_gemm_dW_dX2(X, W_gate, W_val, expert_offset, dg, dv)
        elif ctx.needs_input_grad[0]:
            dX = ext.bwd_grouped_gemm_dX2(W_gate, W_val, expert_offset, dg, dv)
        elif ctx.needs_input_grad[2]:
            dW_gate = ext.bwd_grouped_gemm_dW_kernel(X, expert_offset, dg)
        if ctx.needs_input_grad[3]:
            dW_val = ext.bwd_grouped_gemm_dW_kernel(X, expert_offset, dv)
        return dX, None, dW_gate, dW_val, dW_out


def swiglu_ffn_fn(X, W_gate, W_val, W_out, expert_offset):
    return SwiGLUFFN_FN.apply(X, expert_offset, W_gate, W_val, W_out)


# --------------------------------------------------------------- layer ops


class DispatchFN(torch.autograd.Function):
    """Fused count + offsets + pack for the layer.

    Forward returns (packed_X, packed_topk_weights, counts, offsets, token_id,
    inv); the integer outputs are non-differentiable. Backward is the pack
    backward driven by the inverse map.
    """

    @staticmethod
    def forward(ctx, X, topk_weights, topk_experts, num_experts, counted_ws=None):
        # counted_ws: the workspace route_count_fn returned for these tokens,
        # already holding the per-block expert counts (the counting pass is
        # then skipped).
        ext = get_hip_extension()
        if counted_ws is None:
            outs = ext.dispatch_tokens(X, topk_weights, topk_experts, num_experts)
        else:
            outs = ext.dispatch_tokens_counted(X, topk_weights, topk_experts, num_experts,
                                               counted_ws)
        counts, offsets, packed_X, token_id, _expert, packed_w, inv = outs
        ctx.save_for_backward(inv)
        ctx.mark_non_differentiable(counts, offsets, token_id, inv)
        # No zero-filled grads for the integer outputs (or an unused packed_w).
        ctx.set_materialize_grads(False)
        return packed_X, packed_w, counts, offsets, token_id, inv

    @staticmethod
    def backward(ctx, packed_X_grad, packed_w_grad, *_):
        ext = get_hip_extension()
        (inv,) = ctx.saved_tensors
        if packed_X_grad is None:
            raise RuntimeError("dispatch_fn backward needs a gradient for packed_X")
        if packed_w_grad is None:
            packed_w_grad = torch.zeros(inv.numel(), dtype=torch.float32, device=inv.device)
        X_grad, w_grad = ext.pack_backward_inv(
            packed_X_grad.contiguous(), packed_w_grad.contiguous(), inv
        )
        return X_grad, w_grad, None, None, None


class CombineInvFN(torch.autograd.Function):
    """Combine by inverse map; output in ``out_dtype`` (float32 on the reference surface).

    Backward accepts the grad in float32 or the activation dtype without a cast
    pass and returns (expert_output_grad, None, packed_topk_weights_grad, None).
    """

    @staticmethod
    def forward(ctx, packed_expert_outputs, inv, packed_topk_weights, out_dtype):
        ext = get_hip_extension()
        out = ext.combine_inv(packed_expert_outputs, inv, packed_topk_weights, out_dtype)
        ctx.save_for_backward(packed_expert_outputs, inv, packed_topk_weights)
        return out

    @staticmethod
    def backward(ctx, grad):
        ext = get_hip_extension()
        y, inv, w = ctx.saved_tensors
        if grad.dtype not in (torch.float32, y.dtype):
            grad = grad.to(torch.float32)
        dy, dw = ext.combine_backward_inv(y, inv, w, grad.contiguous())
        return dy, None, dw, None


class RouteFN(torch.autograd.Function):
    """Fused router gate: logits [T,E] f32 -> (gates [T,k] f32, topk [T,k] int32).

    Top-k by logit with ties to the lower expert id (the top-k of the
    softmax probabilities), gates = the selected probabilities renormalised
    (reference src/model/cuda_backend.py:30-37). Backward returns dlogits.
    """

    @staticmethod
    def forward(ctx, logits, top_k):
        ext = get_hip_extension()
        gates, topk = ext.route_topk(logits.contiguous(), top_k)
        ctx.save_for_backward(gates, topk)
        ctx.num_experts = logits.shape[1]
        ctx.mark_non_differentiable(topk)
        ctx.set_materialize_grads(False)  # no zero-filled grad for the int32 ids
        return gates, topk

    @staticmethod
    def backward(ctx, dgates, _dtopk):
        ext = get_hip_extension()
        gates, topk = ctx.saved_tensors
        if dgates is None:
            return None, None
        return ext.route_topk_backward(gates, topk, dgates.contiguous().float(),
                                       ctx.num_experts), None


class RouteCountFN(torch.autograd.Function):
    """RouteFN with the dispatch's expert count fused into the router kernel.

    Returns (gates, topk, dispatch_ws): dispatch_ws holds the per-block
    expert counts for the tokens X (X fixes the block size and device) and
    goes to dispatch_fn(..., counted_ws=dispatch_ws). Same gates, ids and
    backward as RouteFN.
    """

    @staticmethod
    def forward(ctx, logits, top_k, X):
        ext = get_hip_extension()
        gates, topk, ws = ext.route_topk_count(logits.contiguous(), top_k, X)
        ctx.save_for_backward(gates, topk)
        ctx.num_experts = logits.shape[1]
        ctx.mark_non_differentiable(topk, ws)
        ctx.set_materialize_grads(False)
        return gates, topk, ws

    @staticmethod
    def backward(ctx, dgates, _dtopk, _dws):
        ext = get_hip_extension()
        gates, topk = ctx.saved_tensors
        if dgates is None:
            return None, None, None
        return ext.route_topk_backward(gates, topk, dgates.contiguous().float(),
                                       ctx.num_experts), None, None


class RouteDispatchFN(torch.autograd.Function):
    """Router gate (with the dispatch's count) and dispatch in one Function.

    Forward: route_topk_count on logits [T,E] f32, then dispatch_tokens_counted
    of X with those gates. Returns (gates, topk, packed_X, packed_w, counts,
    offsets, token_id, inv), the outputs of RouteCountFN and DispatchFN.
    Backward: when the gates get no gradient of their own (they feed only the
    dispatch), one launch writes dX and dlogits (pack_backward_inv_route);
    otherwise the pack backward's gate gradient is added to theirs before the
    router's backward. Either way the result equals RouteCountFN followed by
    DispatchFN.
    """

    @staticmethod
    def forward(ctx, logits, top_k, X, num_experts):
        ext = get_hip_extension()
        gates, topk, ws = ext.route_topk_count(logits.contiguous(), top_k, X)
        outs = ext.dispatch_tokens_counted(X, gates, topk, num_experts, ws)
        counts, offsets, packed_X, token_id, _expert, packed_w, inv = outs
        ctx.save_for_backward(gates, topk, inv)
        ctx.num_experts = logits.shape[1]
        ctx.mark_non_differentiable(topk, counts, offsets, token_id, inv)
        ctx.set_materialize_grads(False)
        return gates, topk, packed_X, packed_w, counts, offsets, token_id, inv

    @staticmethod
    def backward(ctx, dgates, _dtopk, packed_X_grad, packed_w_grad, *_):
        ext = get_hip_extension()
        gates, topk, inv = ctx.saved_tensors
        if packed_X_grad is None:
            raise RuntimeError("route_dispatch_fn backward needs a gradient for packed_X")
        if packed_w_grad is None:
            packed_w_grad = torch.zeros(inv.numel(), dtype=torch.float32, device=inv.device)
        dpX, dpw = packed_X_grad.contiguous(), packed_w_grad.contiguous()
        if dgates is None:
            X_grad, dlogits = ext.pack_backward_inv_route(dpX, dpw, inv, gates, topk,
                                                          ctx.num_experts)
        else:
            X_grad, w_grad = ext.pack_backward_inv(dpX, dpw, inv)
            dlogits = ext.route_topk_backward(gates, topk, (w_grad + dgates.float()).contiguous(),
                                              ctx.num_experts)
        return dlogits, None, X_grad, None


class RouterGateFN(torch.autograd.Function):
    """The router's logits x32 @ weight.T (float32) for the gate path.

    x [T,d], x32 the same in float32, weight [E,d] float32, E <= 32. One
    kernel gives dx = dl W in x's dtype and dW = dl^T x (reference
    src/model/cuda_backend.py:27-30). What is saved is x32, as the linear on
    the cast tokens saves it: a 16-bit x may be written to after the forward
    (an in-place residual).
    """

    @staticmethod
    def forward(ctx, x, x32, weight):
        ctx.save_for_backward(x32, weight)
        ctx.x_dtype = x.dtype
        ctx.set_materialize_grads(False)
        return torch.nn.functional.linear(x32, weight)

    @staticmethod
    def backward(ctx, dl):
        x32, weight = ctx.saved_tensors
        need_dx, need_dx32, need_dW = ctx.needs_input_grad
        if dl is None:
            return None, None, None
        if torch.is_grad_enabled():  # differentiated again: torch ops, dx through the cast
            return (None, dl @ weight if need_dx32 else None, dl.t() @ x32 if need_dW else None)
        dx, dW = get_hip_extension().router_linear_backward(
            x32.contiguous(), weight.contiguous(), dl.contiguous(), None, need_dx, need_dW,
            ctx.x_dtype)
        return dx, None, dW


class RouterStatsFN(torch.autograd.Function):
    """Load-balancing statistics of the logits (reference src/model/utils.py:77-93).

    Returns (total, frac [E], mean [E], aux): counts.sum(), counts / total,
    softmax(logits).mean(0) and coef * (frac * mean).sum(); mean and aux carry
    gradients to the logits.
    """

    @staticmethod
    def forward(ctx, logits, counts, coef):
        logits = logits.contiguous()
        total, frac, mean, aux = get_hip_extension().router_stats(logits, counts.contiguous(),
                                                                  coef)
        ctx.save_for_backward(logits, frac)
        ctx.coef = coef
        ctx.mark_non_differentiable(total, frac)
        ctx.set_materialize_grads(False)
        return total, frac, mean, aux

    @staticmethod
    def backward(ctx, _dtotal, _dfrac, dmean, daux):
        logits, frac = ctx.saved_tensors
        if dmean is None and daux is None:
            return None, None, None
        if torch.is_grad_enabled():  # differentiated again: composed of torch ops
            return _stats_dlogits(logits, frac, daux, dmean, ctx.coef), None, None
        return get_hip_extension().router_stats_backward(
            logits, frac, None if daux is None else daux.contiguous(),
            None if dmean is None else dmean.contiguous(), ctx.coef), None, None


def _stats_dlogits(logits, frac, daux, dmean, coef):
    v = 0.0
    if daux is not None:
        v = v + daux * coef * frac
    if dmean is not None:
        v = v + dmean
    v = v / logits.shape[0]
    p = logits.softmax(dim=-1)
    return p * (v - (p * v).sum(dim=-1, keepdim=True))


class RouterAuxFN(torch.autograd.Function):
    """RouterStatsFN on the router's second pass, with the gradient to its weight.

    The reference runs the router twice, the second time on detached tokens
    (src/model/cuda_backend.py:40-41), so that the auxiliary loss reaches only
    the router's weight. Both passes compute the same logits, so the first
    pass's are taken; the graph is the second pass's own (one of the two can
    be differentiated and freed before the other). logits [T,E] float32 =
    x32 @ weight.T, x32 [T,d] float32 and logits without gradients, E <= 32.
    """

    @staticmethod
    def forward(ctx, logits, x32, weight, counts, coef):
        logits = logits.contiguous()
        total, frac, mean, aux = get_hip_extension().router_stats(logits, counts.contiguous(),
                                                                  coef)
        ctx.save_for_backward(logits, frac, x32, weight)
        ctx.coef = coef
        ctx.mark_non_differentiable(total, frac)
        ctx.set_materialize_grads(False)
        return total, frac, mean, aux

    @staticmethod
    def backward(ctx, _dtotal, _dfrac, dmean, daux):
        logits, frac, x32, weight = ctx.saved_tensors
        if dmean is None and daux is None:
            return None, None, None, None, None
        if torch.is_grad_enabled():  # differentiated again: composed of torch ops
            da = _stats_dlogits(x32 @ weight.t(), frac, daux, dmean, ctx.coef)
            return None, None, da.t() @ x32, None, None
        ext = get_hip_extension()
        da = ext.router_stats_backward(logits, frac, None if daux is None else daux.contiguous(),
                                       None if dmean is None else dmean.contiguous(), ctx.coef)
        _, dW = ext.router_linear_backward(x32.contiguous(), weight.contiguous(), None, da,
                                           False, True)
        return None, None, dW, None, None


def router_gate_fn(x, x32, weight):
    return RouterGateFN.apply(x, x32, weight)


def router_aux_fn(logits, x32, weight, counts, coef):
    """Statistics of RouterStatsFN; logits and x32 are used without their gradients."""
    return RouterAuxFN.apply(logits.detach(), x32.detach(), weight, counts, coef)


def router_stats_fn(logits, counts, coef):
    return RouterStatsFN.apply(logits, counts, coef)


def route_fn(logits, top_k):
    return RouteFN.apply(logits, top_k)


def route_count_fn(logits, top_k, X):
    return RouteCountFN.apply(logits, top_k, X)


def route_dispatch_fn(logits, top_k, X, num_experts):
    return RouteDispatchFN.apply(logits, top_k, X, num_experts)


def dispatch_fn(X, topk_weights, topk_experts, num_experts, counted_ws=None):
    return DispatchFN.apply(X, topk_weights, topk_experts, num_experts, counted_ws)


def combine_inv_fn(packed_expert_outputs, inv, packed_topk_weights, out_dtype=torch.float32):
    return CombineInvFN.apply(packed_expert_outputs, inv, packed_topk_weights, out_dtype)


# ------------------------------------------------------------- few tokens


def _tracked(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def moe_few_tokens(x, weights, top_k, router_weight=None, logits=None):
    """A whole MoE layer for the few tokens (at most 64) of a decode step.

    x [T,d]; weights (W_gate, W_val, W_out) for SwiGLU experts or (W_up, W_down) for GELU
    ones; either the router's weight [E,d] or its logits [T,E], float32. Returns (out [T,d],
    gates [T,k] float32, ids [T,k] int32): the values of route_fn, dispatch, the experts'
    grouped GEMMs and combine (reference src/model/cuda_backend.py:17-81), with only the
    hidden values rounded to x's dtype on the way. With ``Int8Weight``s tokens and hidden values
    go to 8 bits row by row. Inference only: it raises where a gradient or a forward-mode tangent
    would be lost.
    """
    if len(weights) not in (2, 3):
        raise RuntimeError("weights are (W_gate, W_val, W_out) or (W_up, W_down)")
    int8 = [isinstance(w, Int8Weight) for w in weights]
    if any(int8) and not all(int8):
        raise RuntimeError("the weights are all in 8 bits or none is")
    if _tracked(x, *(() if int8[0] else weights), router_weight, logits):
        raise RuntimeError("moe_few_tokens has no backward: call it under torch.no_grad()")
    if int8[0]:
        up, val, down = weights[0], weights[1] if len(weights) == 3 else None, weights[-1]
        _check_chain(x, up, val, down)
        return get_hip_extension().int8_moe_few_tokens(
            x, up.codes, up.scale, *((None, None) if val is None else (val.codes, val.scale)),
            down.codes, down.scale, top_k, router_weight, logits)
    return get_hip_extension().moe_few_tokens(
        x, weights[0], weights[1] if len(weights) == 3 else None, weights[-1], top_k,
        router_weight, logits)


# ------------------------------------------------------------ block norms


_NORM_KINDS = {"rms": False, "layer": True}


def _block_norm(x, y, w, b, gate, scale, w_next, b_next, kind, eps, dtype):
    if kind not in _NORM_KINDS:
        raise RuntimeError(f"norm kind {kind!r}: expected 'rms' or 'layer'")
    return get_hip_extension().block_norm_fn(x, y, w, b, gate, scale, w_next, b_next,
                                             _NORM_KINDS[kind], eps, dtype)


def pre_norm_fn(x, weight, bias=None, kind="rms", eps=1e-6, dtype=None):
    """The norm before a block: N(x; weight, bias) over the last dimension, in ``dtype``.

    ``kind`` "rms" (no bias) or "layer"; x float32, float16 or bfloat16, and ``dtype`` x's
    or, for a float32 residual stream, a 16-bit one. Weight and bias [d] share a dtype.
    """
    return _block_norm(x, None, None, None, None, None, weight, bias, kind, eps, dtype)[1]


def post_norm_fn(x, y, weight=None, bias=None, gate=None, scale=None, next_weight=None,
                 next_bias=None, kind="rms", eps=1e-6):
    """After a block with input x and output y: h = x + scale * gate * N(y; weight, bias).

    Without a weight N(y) is y; ``gate`` is of y's shape or one value a row, in y's dtype;
    ``scale`` [d] or one value. With ``next_weight`` the next block's norm of h comes from
    the same pass and (h, n) is returned, else h. x is of y's dtype or float32, h of x's, n
    of y's; the parameters share a dtype and get their gradients in it.
    """
    h, n = _block_norm(x, y, weight, bias, gate, scale, next_weight, next_bias, kind, eps, None)
    return h if next_weight is None else (h, n)


# ------------------------------------------------------ 8-bit checkpoints


def checkpoint8(x):
    """(codes int8 [rows,f], exponents uint8 [rows,ceil(f/32)]) of x's rows.

    32 columns share a power of two; a value is off by at most 1/127.5 of its block's
    largest. A block with an infinity or a NaN decodes to NaN.
    """
    return get_hip_extension().checkpoint8(x)


def checkpoint8_decode(codes, exponents, dtype):
    """The rows that a checkpoint holds (exact in the dtype that was kept)."""
    return get_hip_extension().checkpoint8_decode(codes, exponents, dtype)


def gelu8_fn(h):
    """gelu(h) (erf) of rows [rows,f], h kept in 8 bits: the backward is gelu' at the value kept."""
    return get_hip_extension().gelu8_fn(h)


def swiglu8_fn(gate, value):
    """silu(gate) * value of rows [rows,f], both kept in 8 bits for the backward."""
    return get_hip_extension().swiglu8_fn(gate, value)


def _once_differentiable(backward):
    """Second derivatives through ``backward`` raise.

    Unlike torch's decorator, also where the output's gradient needs none itself (a
    gradient penalty on a plain sum), which would count as a constant there.
    """
    @functools.wraps(backward)
    def run(ctx, *dys):
        with torch.no_grad():
            grads = backward(ctx, *dys)
        if not torch.is_grad_enabled():
            return grads
        what = backward.__qualname__.split(".")[0]
        return tuple(get_hip_extension().once_differentiable(list(grads), list(dys), what))
    return run


class GroupedGeluFFN8_FN(torch.autograd.Function):
    """GroupedGeluFFN_FN that keeps X and h = X W_up in 8 bits instead of X, gelu(h), gelu'(h).

    The forward is grouped_gemm_fn, gelu, grouped_gemm_fn; the backward recomputes gelu and
    gelu' from the h kept and takes the weight gradients from the values kept.
    """

    @staticmethod
    def forward(ctx, X, expert_offset, W_up, W_down):
        ext = get_hip_extension()
        X = X.contiguous()
        act, *kept = ext.gelu_checkpoint8(ext.grouped_gemm_kernel(X, expert_offset, W_up), True)
        kept_X = ext.checkpoint8(X) if ctx.needs_input_grad[2] else (None, None)
        ctx.save_for_backward(expert_offset, W_up, W_down, *kept, *kept_X)
        return ext.grouped_gemm_kernel(act, expert_offset, W_down)

    @staticmethod
    @_once_differentiable
    def backward(ctx, dy):
        ext = get_hip_extension()
        off, W_up, W_down, codes, exps, *kept_X = ctx.saved_tensors
        dy = dy.contiguous()
        need_X, _, need_up, need_down = ctx.needs_input_grad
        dX = dW_up = dW_down = None
        dact = ext.bwd_grouped_gemm_dX_kernel(W_down, off, dy)
        dh, act = ext.gelu_backward8(dact, codes, exps, need_down)
        if need_down:
            dW_down = ext.bwd_grouped_gemm_dW_kernel(act, off, dy)
        if need_up:
            X = ext.checkpoint8_decode(*kept_X, dy.dtype)
            if need_X:
                dW_up, dX = ext.bwd_grouped_gemm_dW_dX(X, W_up, off, dh)
            else:
                dW_up = ext.bwd_grouped_gemm_dW_kernel(X, off, dh)
        elif need_X:
            dX = ext.bwd_grouped_gemm_dX_kernel(W_up, off, dh)
        return dX, None, dW_up, dW_down


class SwiGLUFFN8_FN(torch.autograd.Function):
    """SwiGLUFFN_FN that keeps X, gate and value in 8 bits instead of X, hidden, gate, value."""

    @staticmethod
    def forward(ctx, X, expert_offset, W_gate, W_val, W_out):
        ext = get_hip_extension()
        X = X.contiguous()
        hidden, gate, value = ext.grouped_gemm_swiglu(X, expert_offset, W_gate, W_val)
        need_W = ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
        kept_X = ext.checkpoint8(X) if need_W else (None, None)
        ctx.save_for_backward(expert_offset, W_gate, W_val, W_out, *ext.checkpoint8(gate),
                              *ext.checkpoint8(value), *kept_X)
        del gate, value
        return ext.grouped_gemm_kernel(hidden, expert_offset, W_out)

    @staticmethod
    @_once_differentiable
    def backward(ctx, dy):
        ext = get_hip_extension()
        off, W_gate, W_val, W_out, gc, ge, vc, ve, *kept_X = ctx.saved_tensors
        dy = dy.contiguous()
        need_X, _, need_gate, need_val, need_out = ctx.needs_input_grad
        dX = dW_gate = dW_val = dW_out = None
        dhidden = ext.bwd_grouped_gemm_dX_kernel(W_out, off, dy)
        dg, dv, hidden = ext.swiglu_backward8(dhidden, gc, ge, vc, ve, need_out)
        if need_out:
            dW_out = ext.bwd_grouped_gemm_dW_kernel(hidden, off, dy)
        del hidden, dhidden
        X = ext.checkpoint8_decode(*kept_X, dy.dtype) if need_gate or need_val else None
        if need_X and need_gate:
            dW_gate, dX = ext.bwd_grouped_gemm_dW_dX2(X, W_gate, W_val, off, dg, dv)
        elif need_X:
            dX = ext.bwd_grouped_gemm_dX2(W_gate, W_val, off, dg, dv)
        elif need_gate:
            dW_gate = ext.bwd_grouped_gemm_dW_kernel(X, off, dg)
        if need_val:
            dW_val = ext.bwd_grouped_gemm_dW_kernel(X, off, dv)
        return dX, None, dW_gate, dW_val, dW_out


def grouped_gelu_ffn8_fn(X, W_up, W_down, expert_offset):
    if not _tracked(X, W_up, W_down):
        return grouped_gelu_ffn_fn(X, W_up, W_down, expert_offset)
    return GroupedGeluFFN8_FN.apply(X, expert_offset, W_up, W_down)


def swiglu_ffn8_fn(X, W_gate, W_val, W_out, expert_offset):
    if not _tracked(X, W_gate, W_val, W_out):
        return swiglu_ffn_fn(X, W_gate, W_val, W_out, expert_offset)
    return SwiGLUFFN8_FN.apply(X, expert_offset, W_gate, W_val, W_out)


# ---------------------------------------------------------- 8-bit integers


class Int8Weight(NamedTuple):
    """Weights [E,K,N] in 8-bit integers with a float32 scale for each expert and column.

    codes int8 [E, N/64, K/64, 4, 4, 16, 16] (N padded with zeros to 64, K to 128): element
    [e, n//64, k//64, t, g, i, k%16] with g = k%64 // 16 and n%64 = 16 (i//4) + 4 t + i%4;
    scale [E,N]; shape (E, K, N). ``int8_weight`` makes one.
    """

    codes: torch.Tensor
    scale: torch.Tensor
    shape: tuple[int, int, int]


def int8_weight(W):
    """W [E,K,N] (or [K,N], as one expert) as an Int8Weight: every channel's largest magnitude is 127.

    Each value goes to the nearest multiple of its channel's scale, ties to even. A channel with
    an infinity or a NaN has a NaN scale. W gets no gradient.
    """
    if W.dim() == 2:
        W = W.unsqueeze(0)
    codes, scale = get_hip_extension().int8_weight(W.contiguous())
    return Int8Weight(codes, scale, tuple(W.shape))


def int8_weight_decode(weight, dtype):
    """The weights [E,K,N] that an Int8Weight holds, in ``dtype``."""
    _check_int8(weight)
    return get_hip_extension().int8_weight_decode(weight.codes, weight.scale, weight.shape[1],
                                                  dtype)


def int8_rows(x):
    """(codes int8 [rows/16, f/64, 4, 16, 16], scales float32 [rows]) of x [rows,f].

    Row r's integer for column c is codes[r//16, c//64, c%64 // 16, r%16, c%16]; f is padded with
    zeros to 128, rows past the last hold anything. Times its row's scale it is the value's
    nearest multiple of the row's largest magnitude / 127 (ties to even). A row with an infinity
    or a NaN has a NaN scale. Neither has a gradient.
    """
    return get_hip_extension().int8_rows(x.contiguous())


def int8_rows_decode(codes, scales, width, dtype):
    """The rows [rows, width] that codes and scales hold, in ``dtype``."""
    return get_hip_extension().int8_rows_decode(codes, scales, width, dtype)


def _check_int8(*weights):
    for w in weights:
        if not isinstance(w, Int8Weight):
            raise RuntimeError(f"expected an Int8Weight, got {type(w).__name__}")
        if len(w.shape) != 3 or (w.shape[0], w.shape[2]) != tuple(w.scale.shape):
            raise RuntimeError(f"an Int8Weight of shape {tuple(w.shape)} with scales "
                               f"{tuple(w.scale.shape)}")


def _check_chain(x, up, val, down):
    """Whether x, the up (and value) and the down weights of a feed-forward block fit."""
    _check_int8(up, *(() if val is None else (val,)), down)
    E, d, f = up.shape
    if x.dim() != 2 or x.shape[1] != d or tuple(down.shape) != (E, f, d) or (
            val is not None and tuple(val.shape) != (E, d, f)):
        raise RuntimeError(f"x {tuple(x.shape)} and weights {tuple(up.shape)}, "
                           f"{None if val is None else tuple(val.shape)}, {tuple(down.shape)} "
                           "do not fit")


def _all_rows(x, expert_offset):
    """The offsets of a backward: those given, or one expert's of all rows."""
    if expert_offset is not None:
        return expert_offset
    return torch.arange(2, dtype=torch.int32, device=x.device) * x.shape[0]


def _int8_direct(dout, experts, K):
    """Whether the kernels that read 8-bit weights give dout @ W^T; else the weights go to
    dout's dtype first and to the product of that.

    16-bit gradients of weights rounded to 16 bits: where reading and writing the weights costs
    more than the products gain from weights in 16 bits, at most 512 rows an expert and 2^25
    weights or more (128 experts of 2,048 x 768, 14,312 rows: 93 us against 241; 8 of 4,096 x
    14,336, 1,000 rows: 286 against 486, 8,192 rows: 1,056 against 1,042; 1 of 1,024 x 4,096,
    4,096 rows: 69 against 55).
    float32: where tiles of 128 rows by 256 columns would fill half of the chip (8 of 1,024 x
    2,730, 8,192 rows: 228 us against 286; 1 of 1,024 x 4,096, 4,096 rows: 183 against 243; below,
    8 of 1,024 x 4,096, 2,000 rows: 163 against 160; 7 of 300 x 1,365, 5,003 rows: 72 against 65).
    """
    A, N = dout.shape
    if dout.dtype == torch.float32:
        return (A + 128 * experts) * K >= 1 << 22
    return A <= 512 * experts and experts * K * N >= 1 << 25


def _aligned(t):
    """t's rows, those of 16 bits of a multiple of 8 values (zeros are added) and aligned."""
    if t.shape[1] % 8 and t.dtype != torch.float32:
        return torch.nn.functional.pad(t, (0, -t.shape[1] % 8)).contiguous()
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _int8_dx(dout, off, codes, scale, K, exact):
    """dout @ W^T for the weights [E,K,N] that codes and scale hold."""
    ext = get_hip_extension()
    if exact and dout.dtype != torch.float32:
        return ext.int8_dx(dout.contiguous(), off, codes, scale, K, True)
    if _int8_direct(dout, scale.shape[0], K):
        return ext.int8_dx(_aligned(dout), off, codes, scale, K)
    W = ext.int8_weight_decode(codes, scale, K, dout.dtype)
    return ext.bwd_grouped_gemm_dX_kernel(W, _all_rows(dout, off), dout.contiguous())


class Int8GroupedGEMM_FN(torch.autograd.Function):
    """X by frozen 8-bit weights; the gradient to X is dOut times the weights held, transposed.

    The rounding of X is passed straight through. ``exact``: only the result is rounded to dOut's
    dtype; else 16-bit gradients take the weights in dOut's dtype, which is a rounding as large
    as the output's own, for three fifths of the time.
    """

    @staticmethod
    def forward(ctx, X, expert_offset, weight, exact=True):
        ctx.save_for_backward(expert_offset, weight.codes, weight.scale)
        ctx.shape, ctx.exact = weight.shape, exact
        return get_hip_extension().int8_product(X, expert_offset, weight.codes, weight.scale)

    @staticmethod
    @_once_differentiable
    def backward(ctx, dout):
        off, codes, scale = ctx.saved_tensors
        return _int8_dx(dout, off, codes, scale, ctx.shape[1], ctx.exact), None, None, None


class Int8SwiGLUFFN_FN(torch.autograd.Function):
    """SwiGLU FFN on frozen 8-bit weights, with the gradient to X.

    Keeps gate and value in float32; the rounding of X and of the hidden values is passed
    straight through. ``exact``: only the result is rounded to a 16-bit dtype; else the down
    projection's weights are too, for 6 to 21% less time in the backward.
    """

    @staticmethod
    def forward(ctx, X, expert_offset, W_gate, W_val, W_out, exact=True):
        weights = (W_gate, W_val, W_out)
        held = [t for w in weights for t in (w.codes, w.scale)]
        y, gate, value = get_hip_extension().int8_swiglu_ffn(X, expert_offset, *held, True)
        ctx.save_for_backward(expert_offset, gate, value, *held)
        ctx.shape, ctx.exact = W_gate.shape, exact
        return y

    @staticmethod
    @_once_differentiable
    def backward(ctx, dy):
        ext = get_hip_extension()
        off, gate, value, gc, gs, vc, vs, oc, os = ctx.saved_tensors
        E, d, f = ctx.shape
        dy = dy.contiguous() if ctx.exact else _aligned(dy)
        tg, tv = ext.int8_dx_swiglu(dy, gate, value, off, oc, os, gs, vs, f, ctx.exact)
        dX = ext.int8_dx_terms(tg, tv, off, gc, gs, vc, d, dy.dtype)
        return dX, None, None, None, None, None


class Int8GeluFFN_FN(torch.autograd.Function):
    """GELU FFN on frozen 8-bit weights, as Int8SwiGLUFFN_FN; keeps gelu' in float32."""

    @staticmethod
    def forward(ctx, X, expert_offset, W_up, W_down, exact=True):
        held = [t for w in (W_up, W_down) for t in (w.codes, w.scale)]
        y, slope = get_hip_extension().int8_gelu_ffn(X, expert_offset, *held, True)
        ctx.save_for_backward(expert_offset, slope, *held)
        ctx.shape, ctx.exact = W_up.shape, exact
        return y

    @staticmethod
    @_once_differentiable
    def backward(ctx, dy):
        ext = get_hip_extension()
        off, slope, uc, us, dc, ds = ctx.saved_tensors
        E, d, f = ctx.shape
        dy = dy.contiguous() if ctx.exact else _aligned(dy)
        terms = ext.int8_dx_gelu(dy, slope, off, dc, ds, us, f, ctx.exact)
        dX = ext.int8_dx_terms(terms, None, off, uc, us, None, d, dy.dtype)
        return dX, None, None, None, None


def int8_grouped_gemm_fn(X, weight, expert_offset=None, exact_gradient=True):
    """X [A,K] by 8-bit weights [E,K,N], each row by its expert's: [A,N] in X's dtype.

    The rows of X are brought to 8 bits, the products are exact integer sums, scaled in float32
    and rounded once. Without ``expert_offset`` the weights are one linear layer's (E = 1).
    Weights are frozen; X gets its gradient, that of the weights held, rounded once. With
    ``exact_gradient`` False a 16-bit gradient takes the weights rounded to its type first (past
    its largest value: that), which is faster.
    """
    _check_int8(weight)
    if X.dim() != 2 or X.shape[1] != weight.shape[1]:
        raise RuntimeError(f"X {tuple(X.shape)} does not fit weights {tuple(weight.shape)}")
    X = X.contiguous()
    if _tracked(X):
        return Int8GroupedGEMM_FN.apply(X, expert_offset, weight, exact_gradient)
    return get_hip_extension().int8_product(X, expert_offset, weight.codes, weight.scale)


def int8_swiglu_ffn_fn(X, W_gate, W_val, W_out, expert_offset=None, exact_gradient=True):
    """silu(X W_gate) * (X W_val), then W_out, on 8-bit weights: [A,d] in X's dtype.

    X and the hidden values (from their values in X's dtype) are brought to 8 bits row by row;
    gate and value stay in float32 up to the hidden values. X gets its gradient, rounded once;
    with ``exact_gradient`` False a 16-bit one takes the out projection's weights rounded to its
    type (past its largest value: that), which is faster.
    """
    X = X.contiguous()
    _check_chain(X, W_gate, W_val, W_out)
    if _tracked(X):
        return Int8SwiGLUFFN_FN.apply(X, expert_offset, W_gate, W_val, W_out, exact_gradient)
    return get_hip_extension().int8_swiglu_ffn(
        X, expert_offset, W_gate.codes, W_gate.scale, W_val.codes, W_val.scale, W_out.codes,
        W_out.scale, False)[0]


def int8_gelu_ffn_fn(X, W_up, W_down, expert_offset=None, exact_gradient=True):
    """gelu(X W_up) W_down (erf) on 8-bit weights, as int8_swiglu_ffn_fn."""
    X = X.contiguous()
    _check_chain(X, W_up, None, W_down)
    if _tracked(X):
        return Int8GeluFFN_FN.apply(X, expert_offset, W_up, W_down, exact_gradient)
    return get_hip_extension().int8_gelu_ffn(X, expert_offset, W_up.codes, W_up.scale,
                                             W_down.codes, W_down.scale, False)[0]

"""Differentiable expert routing from softmax or sigmoid scores, with a selection bias and expert groups.

The router of the reference's block (softmax -> top-k -> renormalise, vexact/models/qwen3_moe/modeling_qwen3_moe.py:128-134)
is ``ops.router_topk``; this is the form of models whose experts are balanced by a bias on the selection and picked
from a few groups. Its outputs are what ``fused_moe_forward`` takes.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import ops
from ._autograd import once_differentiable


class _GroupedRouterFunction(torch.autograd.Function):
    """Forward: the rollout's kernel. Backward: the derivative of the renormalised, scaled scores at the selected
    experts; the selection itself and the bias have none."""

    @staticmethod
    def forward(ctx, logits, top_k, score, bias, n_groups, topk_groups, group_top, renorm, scale, out_dtype):
        weights, selected = ops.router_topk_grouped(
            logits, top_k, score=score, bias=bias, n_groups=n_groups, topk_groups=topk_groups, group_top=group_top,
            renorm=renorm, scale=scale, out_dtype=out_dtype)
        ctx.save_for_backward(logits if logits.stride(1) == 1 and logits.stride(0) >= logits.shape[1] else logits.contiguous(), selected)
        ctx.call = (score, renorm, scale)
        ctx.mark_non_differentiable(selected)
        ctx.set_materialize_grads(False)  # no zeros for the gradient that the selection does not have
        return weights, selected

    @staticmethod
    @once_differentiable
    def backward(ctx, d_weights, _):
        if d_weights is None:
            return (None,) * 10
        logits, selected = ctx.saved_tensors
        score, renorm, scale = ctx.call
        return (ops._router_grouped_backward(logits, selected, d_weights, score, renorm, scale), *([None] * 9))


def grouped_topk_router(
    logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None, n_groups: int = 1,
    topk_groups: int = 1, group_top: int = 2, renorm: bool = True, scale: float = 1.0, out_dtype: torch.dtype = torch.bfloat16,
):
    """``(routing_weights [T, k], selected_experts [T, k] int64)`` of ``logits [T, E]`` (see ``ops.router_topk_grouped``);
    the weights are differentiable with respect to the logits."""
    args = (logits, top_k, score, bias, n_groups, topk_groups, group_top, renorm, scale, out_dtype)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _GroupedRouterFunction.apply(*args)
    return ops.router_topk_grouped(logits, top_k, score=score, bias=bias, n_groups=n_groups, topk_groups=topk_groups,
                                   group_top=group_top, renorm=renorm, scale=scale, out_dtype=out_dtype)

"""Per-token log-probabilities; mirrors ``logprobs_from_logits_flash_attn`` of
``vexact/batch_invariant_ops/standalone_logprobs.py:28-55`` (which returns minus the cross-entropy
of flash-attn's Triton kernel: ``logits[i, label] - logsumexp(logits[i])`` in fp32, with that kernel's
backward and its ``inplace_backward`` option)."""

from __future__ import annotations

import torch

from .. import ops
from ._autograd import once_differentiable


class _LogprobsFunction(torch.autograd.Function):
    """Forward: the rollout's kernel (``vx_logprobs``), so a trainer scores tokens with the rollout's bits.
    Backward: ``d_logits = d_out (onehot(label) - softmax(logits))``, one kernel, optionally into the logits."""

    @staticmethod
    def forward(ctx, logits, labels, inplace_backward):
        flat = logits.reshape(-1, logits.shape[-1])
        out = ops.logprobs(flat, labels.reshape(-1))
        ctx.save_for_backward(flat, labels.reshape(-1), out)
        ctx.inplace, ctx.shape = bool(inplace_backward), logits.shape
        return out.reshape(labels.shape)

    @staticmethod
    def backward(ctx, d_out):
        flat, labels, out = ctx.saved_tensors
        x = flat if flat.stride(-1) == 1 else flat.contiguous()
        d = ops.logprobs_backward(x, labels, out, d_out.reshape(-1), inplace=ctx.inplace and x is flat)
        return d.reshape(ctx.shape), None, None


def logprobs_from_logits_flash_attn(
    logits: torch.Tensor, labels: torch.Tensor, inplace_backward: bool = False
) -> torch.Tensor:
    if torch.is_grad_enabled() and logits.requires_grad:
        return _LogprobsFunction.apply(logits, labels, inplace_backward)
    shape = labels.shape
    out = ops.logprobs(logits.reshape(-1, logits.shape[-1]), labels.reshape(-1))
    return out.reshape(shape)


class _HiddenLogprobsFunction(torch.autograd.Function):
    """Log-probabilities without logits in memory, forward and backward (``ops.vocab_logprobs``)."""

    @staticmethod
    def forward(ctx, hidden, weight, labels, temperature):
        flat = hidden if hidden.dim() == 2 else hidden.reshape(-1, hidden.shape[-1])
        x, w, flat_labels, scale = ops._vocab_operands(flat, weight, labels, temperature)
        ops._vocab_backward_bytes(x, w)  # what the backward does not take is refused before it is needed
        out, lse = ops._vocab_forward(x, w, flat_labels, scale)
        # as the kernels take them: nothing to check or copy again
        ctx.save_for_backward(hidden if x is flat else x, w, flat_labels, lse)
        ctx.scale, ctx.hidden_shape = scale, hidden.shape
        return out.reshape(labels.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out):
        x, w, labels, lse = ctx.saved_tensors
        if x.dim() != 2:
            x = x.reshape(-1, x.shape[-1])
        need_hidden, need_weight = ctx.needs_input_grad[:2]
        d_hidden, d_weight = ops._vocab_backward(x, w, labels, lse, d_out, ctx.scale, need_hidden, need_weight)
        return d_hidden.reshape(ctx.hidden_shape) if need_hidden else None, d_weight, None, None


def logprobs_from_hidden(
    hidden: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, temperature: float = 1.0
) -> torch.Tensor:
    """Log-probabilities (fp32, shape of ``labels``) of ``labels`` under ``softmax(hidden @ weight.T / temperature)``:
    what ``logprobs_from_logits_flash_attn`` gives, from the last hidden states ``[..., H]`` and the output projection
    ``weight [V, H]`` (bf16) instead of ``[..., V]`` logits, which at V = 151936 are 0.3 MB a token in bf16. Under
    autograd both operands have gradients; a label outside the vocabulary (padding) gives NaN and has none. The logits are not rounded to
    bf16 on the way, so this is not the rollout's logprob bit for bit: score both sides with the same function where
    that matters (a row's bits do not depend on the batch)."""
    if hidden.shape[:-1] != labels.shape:
        raise ValueError(f"labels must have the shape of hidden's rows, got {tuple(labels.shape)} and {tuple(hidden.shape)}")
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _HiddenLogprobsFunction.apply(hidden, weight, labels, float(temperature))
    return ops.vocab_logprobs(hidden.reshape(-1, hidden.shape[-1]), weight, labels, temperature)[0].reshape(labels.shape)

"""Post-training losses as autograd functions on CUDA tensors: log-probabilities of labels from logits or straight
from hidden states, the paired preference loss and the clipped policy loss with a KL term.

The kernels are those of `native` (which has the formulas); GPT.preference_loss and GPT.policy_loss fuse the same
kernels with the model's backward. These functions serve other heads and losses: each saves its input logits and a
few floats a row, and its backward reads the logits once more and writes their gradient. Gradients of gradients are
not provided, and labels, old and reference log-probabilities and advantages take no gradient.

In a captured CUDA graph, take gradients with torch.autograd.grad, or make sure that no earlier autograd graph of the
same leaves is alive: torch accumulates a leaf's gradient on the stream of the first graph that used it.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import native as nv


def _new(like: torch.Tensor, *shape, dtype=torch.float32) -> torch.Tensor:
    return torch.empty(*shape, device=like.device, dtype=dtype)


def _logits_grad(logits, labels, lse, dlogps, ignore_index):
    d = torch.empty(logits.shape, device=logits.device, dtype=logits.dtype)
    nv.token_logprobs_bwd(logits, labels, lse, dlogps, d, ignore_index=ignore_index)
    return d


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, ignore_index):
        logps, lse = _new(logits, *labels.shape), _new(logits, *labels.shape)
        nv.token_logprobs(logits, labels, logps, lse=lse, ignore_index=ignore_index)
        ctx.save_for_backward(logits, labels, lse)
        ctx.ignore_index = ignore_index
        return logps

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogps):
        logits, labels, lse = ctx.saved_tensors
        return _logits_grad(logits, labels, lse, dlogps.float().contiguous(), ctx.ignore_index), None, None


def token_logprobs(logits: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100) -> torch.Tensor:
    """log softmax(logits)[label] in fp32, 0 (and a zero gradient) where the label is ignore_index or outside the
    vocabulary. logits [M, V] or [B, T, V], bf16, fp16 or fp32; labels int64 of the leading shape."""
    return _TokenLogprobs.apply(logits, labels.contiguous(), ignore_index)


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, ref_logps, ignore_index, options):
        B, T = labels.shape
        lse, coef, loss = _new(logits, B, T), _new(logits, B), _new(logits, 1)
        seq, margins = _new(logits, B), _new(logits, B // 2)
        nv.preference_loss(logits, labels, ref_logps, token_logps=_new(logits, B, T), lse=lse, seq_logps=seq,
                           margins=margins, coef=coef, loss=loss, ignore_index=ignore_index, **options)
        ctx.save_for_backward(logits, labels, lse, coef)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(seq, margins)
        return loss.view(()), seq, margins

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *unused):
        logits, labels, lse, coef = ctx.saved_tensors
        dlogps = (coef * g)[:, None].expand(labels.shape).contiguous()
        return _logits_grad(logits, labels, lse, dlogps, ctx.ignore_index), None, None, None, None


def preference_loss(logits: torch.Tensor, labels: torch.Tensor, ref_logps: torch.Tensor | None = None, *,
                    kind: str = "sigmoid", beta: float = 0.1, label_smoothing: float = 0.0, margin: float = 0.0,
                    average: bool = False, ignore_index: int = -100):
    """(loss, sequence log-probabilities [2P], margins [P]) of native.preference_loss; the loss is differentiable."""
    options = dict(kind=kind, beta=beta, label_smoothing=label_smoothing, margin=margin, average=average)
    return _PreferenceLoss.apply(logits, labels.contiguous(), ref_logps, ignore_index, options)


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, old_logps, advantages, ref_logps, ignore_index, options):
        shape = labels.shape
        logps, lse, coef = _new(logits, *shape), _new(logits, *shape), _new(logits, *shape)
        stats, counts = _new(logits, 4), _new(logits, shape[0], dtype=torch.int32)
        nv.policy_loss(logits, labels, old_logps, advantages, ref_logps, token_logps=logps, counts=counts, stats=stats,
                       lse=lse, coef=coef, ignore_index=ignore_index, **options)
        ctx.save_for_backward(logits, labels, lse, coef)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(stats, logps)
        return stats[0].clone(), stats, logps

    @staticmethod
    @once_differentiable
    def backward(ctx, g, *unused):
        logits, labels, lse, coef = ctx.saved_tensors
        return (_logits_grad(logits, labels, lse, coef * g, ctx.ignore_index),) + (None,) * 6


def policy_loss(logits: torch.Tensor, labels: torch.Tensor, old_logps: torch.Tensor, advantages: torch.Tensor,
                ref_logps: torch.Tensor | None = None, *, clip_low: float = 0.2, clip_high: float = 0.2,
                kl_coef: float = 0.0, by_sequence: bool = False, ignore_index: int = -100):
    """(loss, stats [4], token log-probabilities) of native.policy_loss; the loss is differentiable."""
    options = dict(clip_low=clip_low, clip_high=clip_high, kl_coef=kl_coef, by_sequence=by_sequence)
    return _PolicyLoss.apply(logits, labels.contiguous(), old_logps, advantages, ref_logps, ignore_index, options)


class _LinearLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, labels, ignore_index):
        logps, lse = _new(x, x.shape[0]), _new(x, x.shape[0])
        nv.linear_logprobs(x, w, labels, logps, lse=lse, ignore_index=ignore_index)
        ctx.save_for_backward(x, w, labels, lse)
        ctx.ignore_index = ignore_index
        return logps

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogps):
        x, w, labels, lse = ctx.saved_tensors
        dx, dw = (_new(t, t.shape[0], (t.shape[1] + 7) // 8 * 8, dtype=t.dtype)[:, :t.shape[1]] if need else None
                  for t, need in zip((x, w), ctx.needs_input_grad))
        nv.linear_logprobs_bwd(x, w, labels, lse, dlogps.float().contiguous(), dx, dw, ignore_index=ctx.ignore_index)
        return dx, dw, None, None


def linear_logprobs(x: torch.Tensor, w: torch.Tensor, labels: torch.Tensor, *, ignore_index: int = -100) -> torch.Tensor:
    """log softmax(x @ w^T)[label] [M] in fp32 from hidden states x [M, K] and a vocabulary weight w [V, K] (both bf16),
    without storing the logits; 0 where the label is ignore_index or outside the vocabulary. The backward holds the
    gradient of at most 1 GiB of logits at a time."""
    return _LinearLogprobs.apply(x, w, labels.contiguous(), ignore_index)

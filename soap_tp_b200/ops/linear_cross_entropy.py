"""Softmax cross entropy over a large vocabulary straight from the hidden states, without the logits.

``loss_i = log sum_j exp(h_i . w_j) - h_i . w_{t_i}``.  The head's product, the softmax and the loss are one pass whose logits stay in
the tensor cores' accumulators; for the gradients the softmax of a bounded number of tokens at a time is in memory, in 16 bits.  A head of 128256
words on 32768 tokens would otherwise keep 16 GB of fp32 logits and as much again of their softmax for the backward pass.

On CUDA, bf16 and reduced to one number, the gradients are made together with the loss and the backward pass multiplies them by its
own gradient (which moves nothing where that is one); so a loss whose gradients nobody wants belongs under ``torch.no_grad()``.  In the other
cases the backward pass computes the logits again.

With ``group`` the weight is this rank's equal slice of the vocabulary, in rank order, as ``ColumnParallelLinear`` stores a head:
log-sum-exp and the target's logit are joined over the group, and the gradient of the (replicated) hidden states is summed over it.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.distributed as dist
from torch import Tensor
from torch.autograd.function import once_differentiable

REDUCTIONS = ("none", "sum", "mean")


def _validate(hidden: Tensor, weight: Tensor, targets: Tensor, reduction: str, workspace_bytes: int) -> None:
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {REDUCTIONS}, got {reduction!r}.")
    if hidden.ndim < 1 or weight.ndim != 2:
        raise ValueError(f"hidden must be (..., depth) and weight (words, depth), got {tuple(hidden.shape)} and {tuple(weight.shape)}.")
    if hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"hidden has depth {hidden.shape[-1]} and weight {weight.shape[1]}.")
    if targets.shape != hidden.shape[:-1]:
        raise ValueError(f"targets must have shape {tuple(hidden.shape[:-1])}, got {tuple(targets.shape)}.")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets must be int64 or int32, got {targets.dtype}.")
    if hidden.dtype != weight.dtype:
        raise TypeError(f"hidden and weight must have one dtype, got {hidden.dtype} and {weight.dtype}.")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must not be empty, got {tuple(weight.shape)}.")
    if hidden.device != weight.device or hidden.device != targets.device:
        raise ValueError(f"hidden, weight and targets must be on one device, got {hidden.device}, {weight.device} and {targets.device}.")
    allowed = (torch.bfloat16, torch.float16) if hidden.is_cuda else (torch.bfloat16, torch.float16, torch.float32, torch.float64)
    if hidden.dtype not in allowed:
        raise TypeError(f"on {hidden.device.type} hidden and weight must be one of {allowed}, got {hidden.dtype}.")
    if workspace_bytes < 1:
        raise ValueError(f"workspace_bytes must be positive, got {workspace_bytes}.")
    largest = 2**31 - 1
    if weight.shape[0] > largest or weight.shape[1] > largest or targets.numel() > largest:
        raise ValueError("tokens, words and depth must each be below 2**31.")


def _world(group) -> int:
    return 1 if group is None else dist.get_world_size(group)


def _join(lse: Tensor, picked: Tensor, group) -> None:
    """``lse`` becomes that over all ranks' words, ``picked`` the target's logit on every rank (both in place)."""
    every = [torch.empty_like(lse) for _ in range(_world(group))]
    dist.all_gather(every, lse, group=group)
    dist.all_reduce(picked, group=group)
    lse.copy_(torch.logsumexp(torch.stack(every), dim=0))


def _wide(dtype: torch.dtype) -> torch.dtype:
    return dtype if dtype == torch.float64 else torch.float32


class _HostHead:
    """The same quantities from plain tensor operations (CPU tensors)."""

    def __init__(self, hidden, weight, targets, ignore_index, first_word, vocabulary) -> None:
        self.hidden, self.weight = hidden.to(_wide(hidden.dtype)), weight.to(_wide(weight.dtype))
        self.counts = targets != ignore_index
        if bool((self.counts & ((targets < 0) | (targets >= vocabulary))).any()):
            raise IndexError(f"a target is neither {ignore_index} nor in [0, {vocabulary}).")
        local = targets.to(torch.int64) - first_word
        self.mine = self.counts & (local >= 0) & (local < weight.shape[0])
        self.local = torch.where(self.mine, local, 0).unsqueeze(1)

    def statistics(self):
        logits = self.hidden @ self.weight.t()
        return torch.logsumexp(logits, dim=1), logits.gather(1, self.local).squeeze(1) * self.mine

    def losses(self, lse, picked, reduction):
        losses = torch.where(self.counts, lse - picked, torch.zeros_like(lse))
        counted = self.counts.sum().to(losses.dtype)
        if reduction == "none":
            return losses, counted
        return (losses.sum() if reduction == "sum" else losses.sum() / counted.clamp(min=1)), counted

    def gradients(self, lse, reduction, grad_loss, counted):
        factor = grad_loss.to(lse.dtype).expand(lse.shape)
        if reduction == "mean":
            factor = factor / counted.clamp(min=1)
        factor = torch.where(self.counts, factor, torch.zeros_like(factor)).unsqueeze(1)
        d = (self.hidden @ self.weight.t() - lse.unsqueeze(1)).exp() * factor
        d.scatter_add_(1, self.local, -factor * self.mine.unsqueeze(1).to(factor.dtype))
        return d @ self.weight, d.t() @ self.hidden


def _device_loss(ctx, hidden, weight, targets, reduction, ignore_index, group, workspace_bytes, want_hidden, want_weight):
    """The loss and each counted token's log-sum-exp; where the gradients can come with it they are left in ``ctx.gradients``."""
    from ..engine import decoder

    head = decoder.Head(hidden, weight, targets, ignore_index, ctx.first_word, ctx.vocabulary)
    lse, picked = torch.empty((2, head.tokens), dtype=torch.float32, device=head.device)
    shared = _world(group) > 1
    # bf16 only: fp16 gradients are rounded after the loss's scale, which the backward pass brings, has been multiplied in
    if (want_hidden or want_weight) and reduction != "none" and head.dtype == torch.bfloat16:
        gradients = decoder.HeadGradients(head, want_hidden, want_weight, workspace_bytes)
        head.prepare(gradients.hidden)
        gradients.factors(reduction, None)
        parts = head.parts(gradients.rows)
        for first, rows in gradients.turns():
            head.statistics(first, rows, parts, lse, picked, gradients.logits)
            if shared:
                _join(lse[first:first + rows], picked[first:first + rows], group)
            gradients.add(first, rows, lse, parts, picked)
        ctx.gradients = (gradients.hidden, gradients.weight)
    else:
        head.prepare()
        head.statistics(0, head.tokens, head.parts(head.tokens), lse, picked)
        if shared:
            _join(lse, picked, group)
    return head.loss(lse, picked, reduction), lse


def _device_gradients(ctx, grad_loss, hidden, weight, targets, lse, want_hidden, want_weight):
    from ..engine import decoder

    head = decoder.Head(hidden, weight, targets, ctx.ignore_index, ctx.first_word, ctx.vocabulary)
    gradients = decoder.HeadGradients(head, want_hidden, want_weight, ctx.workspace_bytes)
    head.prepare(gradients.hidden)
    gradients.factors(ctx.reduction, grad_loss.to(torch.float32).contiguous())
    for first, rows in gradients.turns():
        gradients.add(first, rows, lse)
    return gradients.hidden, gradients.weight


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, reduction, ignore_index, group, workspace_bytes):
        words = weight.shape[0]
        ctx.first_word = 0 if group is None else dist.get_rank(group) * words
        ctx.vocabulary = words * _world(group)
        ctx.reduction, ctx.ignore_index, ctx.group, ctx.workspace_bytes = reduction, ignore_index, group, workspace_bytes
        ctx.gradients = None
        shape = targets.shape
        hidden, targets = hidden.detach().reshape(-1, hidden.shape[-1]), targets.reshape(-1)
        if hidden.is_cuda:
            with torch.cuda.device(hidden.device):
                ctx.captured = torch.cuda.is_current_stream_capturing()
                loss, lse = _device_loss(ctx, hidden, weight, targets, reduction, ignore_index, group, workspace_bytes,
                                         *ctx.needs_input_grad[:2])
            counted = None
        else:
            head = _HostHead(hidden, weight, targets, ignore_index, ctx.first_word, ctx.vocabulary)
            lse, picked = head.statistics()
            if _world(group) > 1:
                _join(lse, picked, group)
            loss, counted = head.losses(lse, picked, reduction)
        ctx.save_for_backward(hidden, weight, targets, lse, counted)
        ctx.shape = (*shape, hidden.shape[-1])
        return loss.view(shape) if reduction == "none" else loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_loss):
        hidden, weight, targets, lse, counted = ctx.saved_tensors
        want_hidden, want_weight = ctx.needs_input_grad[:2]
        if hidden.is_cuda:
            with torch.cuda.device(hidden.device):
                made, ctx.gradients = ctx.gradients, None
                # handed over once: they are the caller's from then on.  A graph of the backward pass alone would scale them again at every replay.
                if made is not None and ctx.captured == torch.cuda.is_current_stream_capturing():
                    from ..engine import decoder

                    decoder.scale_gradients(grad_loss.to(torch.float32), *made)
                    d_hidden, d_weight = made
                else:
                    d_hidden, d_weight = _device_gradients(ctx, grad_loss, hidden, weight, targets, lse, want_hidden, want_weight)
        else:
            head = _HostHead(hidden, weight, targets, ctx.ignore_index, ctx.first_word, ctx.vocabulary)
            d_hidden, d_weight = (g.to(hidden.dtype) for g in head.gradients(lse, ctx.reduction, grad_loss.reshape(-1) if
                                                                             ctx.reduction == "none" else grad_loss, counted))
        if want_hidden and _world(ctx.group) > 1:
            dist.all_reduce(d_hidden, group=ctx.group)
        return d_hidden.view(ctx.shape) if want_hidden else None, d_weight if want_weight else None, None, None, None, None, None


def linear_cross_entropy(
    hidden: Tensor,
    weight: Tensor,
    targets: Tensor,
    *,
    reduction: str = "mean",
    ignore_index: int = -100,
    group: Optional[dist.ProcessGroup] = None,
    workspace_bytes: int = 2**31,
) -> Tensor:
    """Cross entropy of ``softmax(hidden @ weight.T)`` against ``targets``, in fp32 (fp64 for fp64 CPU tensors).

    ``hidden`` (..., depth) and ``weight`` (words, depth) are bf16 or fp16 on CUDA; ``targets`` (...) counts over the whole
    vocabulary.  Tokens whose target is ``ignore_index`` have loss 0 and no gradient; ``"mean"`` is over the others, and 0 where there
    are none.  Another target outside the vocabulary is an error on CPU and makes the loss NaN on CUDA, where nobody waits for
    the device to find out.  ``group``: see the module's text.  The backward pass holds up to ``workspace_bytes`` of softmax
    (256 tokens' at least) and, where the tokens need more than one turn, the weight's gradient in fp32.
    """
    _validate(hidden, weight, targets, reduction, workspace_bytes)
    if targets.numel() == 0:
        loss = (hidden.sum() + weight[:0].sum()).to(_wide(hidden.dtype))
        return loss.expand(targets.shape) if reduction == "none" else loss
    return _LinearCrossEntropy.apply(hidden, weight, targets, reduction, ignore_index, group, workspace_bytes)


__all__ = ["linear_cross_entropy"]

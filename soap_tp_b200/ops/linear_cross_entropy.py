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

import functools
from typing import Optional

import torch
import torch.distributed as dist
from torch import Tensor
from torch.autograd.function import once_differentiable

REDUCTIONS = ("none", "sum", "mean")


_ON_CUDA = (torch.bfloat16, torch.float16)
_ON_CPU = (torch.bfloat16, torch.float16, torch.float32, torch.float64)


@functools.cache
def _native():
    from ..engine import decoder

    return decoder


def _validate(hidden: Tensor, weight: Tensor, targets: Tensor, reduction: str, workspace_bytes: int) -> None:
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction must be one of {REDUCTIONS}, got {reduction!r}.")
    shape, words = hidden.shape, weight.shape
    if len(shape) < 1 or len(words) != 2:
        raise ValueError(f"hidden must be (..., depth) and weight (words, depth), got {tuple(shape)} and {tuple(words)}.")
    if shape[-1] != words[1]:
        raise ValueError(f"hidden has depth {shape[-1]} and weight {words[1]}.")
    if targets.shape != shape[:-1]:
        raise ValueError(f"targets must have shape {tuple(shape[:-1])}, got {tuple(targets.shape)}.")
    if targets.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"targets must be int64 or int32, got {targets.dtype}.")
    if hidden.dtype != weight.dtype:
        raise TypeError(f"hidden and weight must have one dtype, got {hidden.dtype} and {weight.dtype}.")
    if words[0] < 1 or words[1] < 1:
        raise ValueError(f"weight must not be empty, got {tuple(words)}.")
    device = hidden.device
    if device != weight.device or device != targets.device:
        raise ValueError(f"hidden, weight and targets must be on one device, got {device}, {weight.device} and {targets.device}.")
    allowed = _ON_CUDA if hidden.is_cuda else _ON_CPU
    if hidden.dtype not in allowed:
        raise TypeError(f"on {device.type} hidden and weight must be one of {allowed}, got {hidden.dtype}.")
    if workspace_bytes < 1:
        raise ValueError(f"workspace_bytes must be positive, got {workspace_bytes}.")
    if max(words[0], words[1], targets.numel()) >= 2**31:
        raise ValueError("tokens, words and depth must each be below 2**31.")


def _world(group) -> int:
    return 1 if group is None else dist.get_world_size(group)


def _finish(rest: Tensor, picked: Tensor):
    """Log-sum-exp and loss from the log-sum-exp of all words but the target and the target's logit.  (Not their difference: of the loss of
    a token that the model knows nothing would be left.)"""
    over = rest - picked
    by = torch.log1p(torch.exp(-over.abs()))
    return torch.where(over > 0, rest + by, picked + by), torch.where(over > 0, over + by, by)


def _join(group, lse: Tensor, loss: Tensor) -> None:
    """From this rank's log-sum-exp of its words but the target and the target's logit (0 where it has it not) to those of all ranks' words and
    the loss, in place."""
    most = lse.clone()
    dist.all_reduce(most, op=dist.ReduceOp.MAX, group=group)
    most = torch.where(most == float("-inf"), torch.zeros_like(most), most)
    sums = torch.stack(((lse - most).exp(), loss))
    dist.all_reduce(sums, group=group)
    for to, value in zip((lse, loss), _finish(most + sums[0].log(), sums[1])):
        to.copy_(value)


def _wide(dtype: torch.dtype) -> torch.dtype:
    return dtype if dtype == torch.float64 else torch.float32


class _HostHead:
    """The same quantities from plain tensor operations (CPU tensors)."""

    def __init__(self, hidden, weight, targets, ignore_index, first_word, vocabulary) -> None:
        self.counts = targets != ignore_index
        self.hidden, self.weight = hidden.to(_wide(hidden.dtype)), weight.to(_wide(weight.dtype))
        # (what padding holds, NaN included, reaches nothing: zero times it would)
        self.hidden = torch.where(self.counts.unsqueeze(1), self.hidden, torch.zeros_like(self.hidden[:1]))
        if bool((self.counts & ((targets < 0) | (targets >= vocabulary))).any()):
            raise IndexError(f"a target is neither {ignore_index} nor in [0, {vocabulary}).")
        local = targets.to(torch.int64) - first_word
        self.mine = self.counts & (local >= 0) & (local < weight.shape[0])
        self.local = torch.where(self.mine, local, 0).unsqueeze(1)

    def statistics(self):
        """Log-sum-exp of these words but the target, and the target's logit (0 where it is elsewhere)."""
        logits = self.hidden @ self.weight.t()
        picked = logits.gather(1, self.local).squeeze(1) * self.mine
        logits.scatter_(1, self.local, torch.where(self.mine.unsqueeze(1), float("-inf"), logits.gather(1, self.local)))
        return torch.logsumexp(logits, dim=1), picked

    def losses(self, losses, reduction):
        losses = torch.where(self.counts, losses, torch.zeros_like(losses))
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


def _without_autocast(function):
    """The loss is computed in 32 bits at least, whatever autocast is around either pass."""

    @functools.wraps(function)
    def call(*args):
        with torch.autocast("cpu", enabled=False):
            return function(*args)

    return call


class _LinearCrossEntropy(torch.autograd.Function):
    """CPU tensors."""

    @staticmethod
    @_without_autocast
    def forward(ctx, hidden, weight, targets, reduction, ignore_index, group):
        words, world = weight.shape[0], _world(group)
        first_word = 0 if group is None else dist.get_rank(group) * words
        ctx.arguments = (ignore_index, first_word, words * world)
        ctx.reduction, ctx.shape = reduction, hidden.shape
        shape = targets.shape
        hidden, targets = hidden.detach().reshape(-1, hidden.shape[-1]), targets.reshape(-1)
        head = _HostHead(hidden, weight, targets, *ctx.arguments)
        lse, losses = head.statistics()
        if world > 1:
            _join(group, lse, losses)
        else:
            lse, losses = _finish(lse, losses)
        loss, counted = head.losses(losses, reduction)
        ctx.save_for_backward(hidden, weight, targets, lse, counted)
        return loss.view(shape) if reduction == "none" else loss

    @staticmethod
    @once_differentiable
    @_without_autocast
    def backward(ctx, grad_loss):
        hidden, weight, targets, lse, counted = ctx.saved_tensors
        head = _HostHead(hidden, weight, targets, *ctx.arguments)
        if ctx.reduction == "none":
            grad_loss = grad_loss.reshape(-1)
        d_hidden, d_weight = (g.to(hidden.dtype) for g in head.gradients(lse, ctx.reduction, grad_loss, counted))
        wanted = ctx.needs_input_grad
        return d_hidden.view(ctx.shape) if wanted[0] else None, d_weight if wanted[1] else None, None, None, None, None


class _SumGradient(torch.autograd.Function):
    """Hidden states that every rank of a group has: each rank's words give a part of their gradient."""

    @staticmethod
    def forward(ctx, hidden, group):
        ctx.group = group
        return hidden.view_as(hidden)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        grad = grad.contiguous()
        dist.all_reduce(grad, group=ctx.group)
        return grad, None


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
    the device to find out.  On CUDA a token's loss is the same whatever padding surrounds it; it changes by roundings where more than 64
    tokens count (of fewer, logits are rounded to fp32 more often), its gradients where the call has more than 256 tokens (of fewer, the logits'
    gradient has two 16-bit terms).  ``group``: see the module's text.  Up to ``workspace_bytes`` of softmax are in memory at a time
    (256 tokens' at least) and, where the tokens need more than one turn, the weight's gradient in fp32.
    """
    _validate(hidden, weight, targets, reduction, workspace_bytes)
    if targets.numel() == 0:
        loss = (hidden.sum() + weight[:0].sum()).to(_wide(hidden.dtype))
        return loss.expand(targets.shape) if reduction == "none" else loss
    world = _world(group)
    if world > 1:
        hidden = _SumGradient.apply(hidden, group)
    if not hidden.is_cuda:
        return _LinearCrossEntropy.apply(hidden, weight, targets, reduction, ignore_index, group)
    decoder, words = _native(), weight.shape[0]
    return decoder.native.linear_cross_entropy(
        hidden, weight, targets, decoder.REDUCTIONS[reduction], ignore_index, 0 if group is None else dist.get_rank(group) * words, words * world,
        workspace_bytes, decoder.status(hidden.device), functools.partial(_join, group) if world > 1 else None)


__all__ = ["linear_cross_entropy"]

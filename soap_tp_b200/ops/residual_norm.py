"""Norms before and after a block, its gate and its residual scale, as one operator.

A pre-norm decoder alternates ``x = x + block(norm(x))``: every residual sum is followed by the next block's norm, and some decoders put a
norm, a learnt gate or a depth-dependent scale between a block's output and the sum.  :func:`residual_norm` takes all of that in one pass
over memory, forward and backward; :func:`rms_norm` is the norm alone.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

LONGEST_ROW = 32768


def _validate(x: Tensor, branch: Optional[Tensor], vectors: dict, scale: float, eps: float) -> None:
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be (..., dim), got {tuple(x.shape)}.")
    allowed = (torch.bfloat16, torch.float16, torch.float32) + (() if x.is_cuda else (torch.float64,))
    if x.dtype not in allowed:
        raise TypeError(f"on {x.device.type} x must be one of {allowed}, got {x.dtype}.")
    if x.is_cuda and x.shape[-1] > LONGEST_ROW:
        raise ValueError(f"rows of more than {LONGEST_ROW} values are not supported on CUDA, got {x.shape[-1]}.")
    if branch is not None and (branch.shape != x.shape or branch.dtype != x.dtype or branch.device != x.device):
        raise ValueError(f"branch must match x: {tuple(x.shape)} {x.dtype} {x.device}, got {tuple(branch.shape)} {branch.dtype} {branch.device}.")
    given = {name: v for name, v in vectors.items() if v is not None}
    for name, v in given.items():
        if v.shape != x.shape[-1:] or v.device != x.device:
            raise ValueError(f"{name} must have shape {tuple(x.shape[-1:])} on {x.device}, got {tuple(v.shape)} on {v.device}.")
        if v.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must be {x.dtype} or float32, got {v.dtype}.")
    if len({v.dtype for v in given.values()}) > 1:
        raise TypeError(f"{', '.join(given)} must have one dtype, got {[v.dtype for v in given.values()]}.")
    if branch is None and any(given.get(name) is not None for name in ("branch_weight", "gate")):
        raise ValueError("branch_weight and gate need a branch.")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}.")
    if not scale - scale == 0.0:
        raise ValueError(f"scale must be finite, got {scale}.")


def _host_forward(x, branch, weight, branch_weight, gate, scale, eps):
    """The definition in plain tensor operations (CPU tensors; autograd differentiates it)."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32

    def norm(v, w):
        return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps) * w.to(wide)

    h = x.to(wide)
    if branch is not None:
        b = branch.to(wide)
        if branch_weight is not None:
            b = norm(b, branch_weight)
        if gate is not None:
            b = b * gate.to(wide)
        h = h + scale * b
    return x if branch is None else h.to(x.dtype), None if weight is None else norm(h, weight).to(x.dtype)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, weight, branch_weight, gate, scale, eps):
        from ..engine import decoder

        with torch.cuda.device(x.device):
            h, y, rms, branch_rms = decoder.residual_norm_forward(x, branch, weight, branch_weight, gate, scale, eps)
        ctx.save_for_backward(h, branch if branch_weight is not None or gate is not None else None, weight, branch_weight, gate, rms,
                              branch_rms)
        ctx.scale, ctx.eps = scale, eps
        ctx.with_branch = branch is not None
        ctx.set_materialize_grads(False)
        return (h if branch is not None else None), y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_h, grad_y):
        h, branch, weight, branch_weight, gate, rms, branch_rms = ctx.saved_tensors
        if grad_h is None and grad_y is None:
            return (None,) * 7
        from ..engine import decoder

        with torch.cuda.device(h.device):
            want = list(ctx.needs_input_grad[:5])
            # (a branch that is only added is not read again: h stands for its place)
            grads = decoder.residual_norm_backward(h, branch if branch is not None else (h if ctx.with_branch else None), weight, branch_weight,
                                                   gate, ctx.scale, ctx.eps, rms, branch_rms, grad_h, grad_y, want)
        if grad_y is None:
            grads = (*grads[:2], None, *grads[3:])
        return (*grads, None, None)


def residual_norm(
    x: Tensor,
    branch: Tensor,
    weight: Optional[Tensor] = None,
    *,
    branch_weight: Optional[Tensor] = None,
    gate: Optional[Tensor] = None,
    scale: float = 1.0,
    eps: float = 1e-5,
) -> Tuple[Tensor, Optional[Tensor]]:
    """``h = x + scale * gate * norm(branch) * branch_weight`` and ``y = norm(h) * weight``, ``norm(v) = v / sqrt(mean(v^2) + eps)``
    over the last dimension.

    Without ``branch_weight`` the branch has no norm, without ``gate`` no gate; without ``weight`` there is no second norm and ``y`` is None.
    The vectors have ``x``'s dtype or are fp32.  Means, sums and the vectors' gradients are held in fp32; ``h`` and ``y`` are each
    rounded once.  Differentiable once.
    """
    _validate(x, branch, dict(weight=weight, branch_weight=branch_weight, gate=gate), scale, eps)
    if branch is None:
        raise ValueError("residual_norm needs a branch; rms_norm is the norm alone.")
    if not x.is_cuda or x.numel() == 0:
        return _host_forward(x, branch, weight, branch_weight, gate, scale, eps)
    dim = x.shape[-1]
    vectors = [None if v is None else v.contiguous() for v in (weight, branch_weight, gate)]
    h, y = _ResidualNorm.apply(x.reshape(-1, dim), branch.reshape(-1, dim), *vectors, float(scale), float(eps))
    return h.view(x.shape), None if y is None else y.view(x.shape)


def rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-5) -> Tensor:
    """``norm(x) * weight`` as :func:`residual_norm` computes its ``y``."""
    _validate(x, None, dict(weight=weight), 1.0, eps)
    if not x.is_cuda or x.numel() == 0:
        return _host_forward(x, None, weight, None, None, 1.0, eps)[1]
    _, y = _ResidualNorm.apply(x.reshape(-1, x.shape[-1]), None, weight.contiguous(), None, None, 1.0, float(eps))
    return y.view(x.shape)


__all__ = ["residual_norm", "rms_norm"]

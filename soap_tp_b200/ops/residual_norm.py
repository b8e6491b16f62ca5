"""Norms before and after a block, its gate and its residual scale, as one operator.

A pre-norm decoder alternates ``x = x + block(norm(x))``: every residual sum is followed by the next block's norm, and some decoders put a
norm, a learnt gate or a depth-dependent scale between a block's output and the sum.  :func:`residual_norm` takes all of that in one pass
over memory, forward and backward; :func:`rms_norm` is the norm alone.
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch
from torch import Tensor

LONGEST_ROW = 32768
_ON_CUDA = (torch.bfloat16, torch.float16, torch.float32)
_ON_CPU = (*_ON_CUDA, torch.float64)


@functools.cache
def _native():
    from ..engine import decoder

    return decoder


def _validate(x: Tensor, branch: Optional[Tensor], weight: Optional[Tensor], branch_weight: Optional[Tensor], gate: Optional[Tensor],
              scale: float, eps: float) -> None:
    shape, dtype, device = x.shape, x.dtype, x.device
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"x must be (..., dim), got {tuple(shape)}.")
    allowed = _ON_CUDA if x.is_cuda else _ON_CPU
    if dtype not in allowed:
        raise TypeError(f"on {device.type} x must be one of {allowed}, got {dtype}.")
    if shape[-1] > LONGEST_ROW and x.is_cuda:
        raise ValueError(f"rows of more than {LONGEST_ROW} values are not supported on CUDA, got {shape[-1]}.")
    if branch is not None and (branch.shape != shape or branch.dtype != dtype or branch.device != device):
        raise ValueError(f"branch must match x: {tuple(shape)} {dtype} {device}, got {tuple(branch.shape)} {branch.dtype} {branch.device}.")
    common = None
    for name, v in (("weight", weight), ("branch_weight", branch_weight), ("gate", gate)):
        if v is None:
            continue
        if v.shape != shape[-1:] or v.device != device:
            raise ValueError(f"{name} must have shape {tuple(shape[-1:])} on {device}, got {tuple(v.shape)} on {v.device}.")
        if v.dtype != dtype and v.dtype != torch.float32:
            raise TypeError(f"{name} must be {dtype} or float32, got {v.dtype}.")
        if common is not None and v.dtype != common:
            raise TypeError(f"weight, branch_weight and gate must have one dtype, got {common} and {v.dtype}.")
        common = v.dtype
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
    rounded once.  The backward pass keeps x, the branch and two numbers a row.  Differentiable once.
    """
    if branch is None:
        raise ValueError("residual_norm needs a branch; rms_norm is the norm alone.")
    _validate(x, branch, weight, branch_weight, gate, scale, eps)
    if not x.is_cuda or x.numel() == 0:
        return _host_forward(x, branch, weight, branch_weight, gate, scale, eps)
    decoder = _native()
    out = decoder.native.residual_norm(x, branch, weight, branch_weight, gate, scale, eps, decoder.status(x.device))
    return out[0], out[1] if weight is not None else None


def rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-5) -> Tensor:
    """``norm(x) * weight`` as :func:`residual_norm` computes its ``y``."""
    if weight is None:
        raise ValueError("rms_norm needs a weight.")
    _validate(x, None, weight, None, None, 1.0, eps)
    if not x.is_cuda or x.numel() == 0:
        return _host_forward(x, None, weight, None, None, 1.0, eps)[1]
    decoder = _native()
    return decoder.native.residual_norm(x, None, weight, None, None, 1.0, eps, decoder.status(x.device))[0]


__all__ = ["residual_norm", "rms_norm"]

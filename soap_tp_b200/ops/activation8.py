"""Activations kept in 8 bits for the backward pass.

``x`` is kept as whole numbers ``q = round(x / scale)`` with ``scale = max|x| / 127`` over 64 neighbouring features of a row: 8.5 bits a value, off by
``max|x| / 254`` at most.  A group that holds an infinity or a NaN comes back as NaN.

* :func:`pack8`, :func:`unpack8`: the form itself;
* :func:`checkpoint8`: a block that keeps its input this way and is run again from it in the backward pass;
* :func:`swiglu8`: ``silu(gate) * up`` whose backward pass works from gate and up kept this way;
* :func:`swiglu_linear8`: the same with the linear layer behind it, whose input is not kept at all.

Results of the forward pass are those of exact activations; gradients are those of the kept ones.
"""
from __future__ import annotations

from typing import Callable, Iterable, NamedTuple, Tuple

import torch
import torch.nn.functional as F
from torch import Tensor
from torch.autograd.function import once_differentiable

GROUP = 64
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
SMALLEST_SCALE = 2.0 ** -126


class Packed8(NamedTuple):
    """A tensor kept in 8 bits: what :func:`unpack8` needs."""

    values: Tensor            # int8 (rows, features rounded up to 8)
    scales: Tensor            # fp32 (rows, groups of 64 features)
    shape: torch.Size
    dtype: torch.dtype

    def bytes(self) -> int:
        return self.values.numel() + 4 * self.scales.numel()


def _check_values(name: str, x: Tensor) -> None:
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} must be (..., features), got {tuple(x.shape)}.")
    if x.dtype not in DTYPES:
        raise TypeError(f"{name} must be one of {DTYPES}, got {x.dtype}.")


def _host_pack(x: Tensor) -> Tuple[Tensor, Tensor]:
    rows, dim = x.shape
    groups = -(-dim // GROUP)
    v = F.pad(x.float(), (0, groups * GROUP - dim)).view(rows, groups, GROUP)
    scales = (v.abs().amax(dim=2) / 127.0).clamp(min=SMALLEST_SCALE)
    scales = torch.where(torch.isfinite(v).all(dim=2), scales, torch.full_like(scales, float("nan")))
    values = torch.nan_to_num(torch.round(v / scales.unsqueeze(2)), nan=0.0).to(torch.int8).view(rows, groups * GROUP)
    return values[:, : -(-dim // 8) * 8].contiguous(), scales


def _host_unpack(values: Tensor, scales: Tensor, dim: int, dtype: torch.dtype) -> Tensor:
    return (values[:, :dim].float() * scales.repeat_interleave(GROUP, dim=1)[:, :dim]).to(dtype)


def _pack(x: Tensor) -> Tuple[Tensor, Tensor]:
    if x.is_cuda and x.numel() > 0:
        from ..engine import decoder

        with torch.cuda.device(x.device):
            return decoder.pack8(x)
    return _host_pack(x)


def _unpack(values: Tensor, scales: Tensor, dim: int, dtype: torch.dtype) -> Tensor:
    if values.is_cuda and values.numel() > 0:
        from ..engine import decoder

        with torch.cuda.device(values.device):
            return decoder.unpack8(decoder.Kept8(values, scales), dim, dtype)
    return _host_unpack(values, scales, dim, dtype)


@torch.no_grad()
def pack8(x: Tensor) -> Packed8:
    """``x`` (..., features) in 8 bits."""
    _check_values("x", x)
    return Packed8(*_pack(x.reshape(-1, x.shape[-1])), x.shape, x.dtype)


@torch.no_grad()
def unpack8(packed: Packed8) -> Tensor:
    """The values that ``packed`` stands for, in the dtype it was made from."""
    rows, dim = packed.values.shape[0], packed.shape[-1]
    groups = -(-dim // GROUP)
    if packed.shape.numel() != rows * dim or packed.values.shape != (rows, -(-dim // 8) * 8) or packed.scales.shape != (rows, groups):
        raise ValueError(f"values {tuple(packed.values.shape)} and scales {tuple(packed.scales.shape)} do not hold a tensor of shape {tuple(packed.shape)}.")
    if packed.values.dtype != torch.int8 or packed.scales.dtype != torch.float32 or packed.dtype not in DTYPES:
        raise TypeError(f"values are int8 and scales float32, got {packed.values.dtype} and {packed.scales.dtype} for {packed.dtype}.")
    if packed.values.device != packed.scales.device:
        raise ValueError(f"values and scales must be on one device, got {packed.values.device} and {packed.scales.device}.")
    return _unpack(packed.values.contiguous(), packed.scales.contiguous(), dim, packed.dtype).view(packed.shape)


class _Checkpoint8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, function, count, x, *rest):
        ctx.function, ctx.count = function, count
        ctx.shape, ctx.dtype = x.shape, x.dtype
        packed = pack8(x)
        ctx.tensors = [isinstance(a, Tensor) for a in rest]
        ctx.plain = [None if t else a for a, t in zip(rest, ctx.tensors)]
        ctx.save_for_backward(packed.values, packed.scales, *(a for a, t in zip(rest, ctx.tensors) if t))
        with torch.no_grad():
            return function(x, *rest[:count])

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        values, scales, *saved = ctx.saved_tensors
        x = unpack8(Packed8(values, scales, ctx.shape, ctx.dtype)).requires_grad_(ctx.needs_input_grad[2])
        saved = iter(saved)
        rest = [next(saved) if t else a for a, t in zip(ctx.plain, ctx.tensors)]
        # arguments become leaves of the second run; parameters are leaves that the function holds itself
        arguments = [a.detach().requires_grad_(n) if isinstance(a, Tensor) else a
                     for a, n in zip(rest[: ctx.count], ctx.needs_input_grad[3:])]
        wanted = [a for a, n in zip([x, *arguments, *rest[ctx.count:]], ctx.needs_input_grad[2:]) if n]
        with torch.enable_grad():
            outputs = ctx.function(x, *arguments)
        outputs = (outputs,) if isinstance(outputs, Tensor) else tuple(outputs)
        pairs = [(o, g) for o, g in zip(outputs, grads) if isinstance(o, Tensor) and o.requires_grad and g is not None]
        found = iter(torch.autograd.grad([o for o, _ in pairs], wanted, [g for _, g in pairs], allow_unused=True) if pairs and wanted
                     else [None] * len(wanted))
        return (None, None, *(next(found) if n else None for n in ctx.needs_input_grad[2:]))


def checkpoint8(function: Callable, x: Tensor, *args, parameters: Iterable[Tensor] = None):
    """``function(x, *args)`` that keeps nothing but ``x`` in 8 bits (and ``args``, as they are) and is run again, from the kept ``x``, in
    the backward pass.

    ``function`` takes tensors or anything else, returns a tensor or a tuple of tensors, and does the same on every call (it must not
    draw random numbers).  Gradients reach ``x``, tensor ``args`` and ``parameters``: by default those of ``function`` where it is a module.
    Without gradients it is a plain call.
    """
    _check_values("x", x)
    if parameters is None:
        parameters = function.parameters() if isinstance(function, torch.nn.Module) else ()
    parameters = [p for p in parameters if p.requires_grad]
    if not torch.is_grad_enabled() or not any(isinstance(a, Tensor) and a.requires_grad for a in (x, *args, *parameters)):
        return function(x, *args)
    return _Checkpoint8.apply(function, len(args), x, *args, *parameters)


def _check_swiglu(gate: Tensor, up: Tensor) -> None:
    _check_values("gate", gate)
    if gate.shape != up.shape or gate.dtype != up.dtype or gate.device != up.device:
        raise ValueError(f"gate and up must match, got {tuple(gate.shape)} {gate.dtype} {gate.device} and {tuple(up.shape)} {up.dtype} {up.device}.")


def _swiglu_forward(gate: Tensor, up: Tensor, keep: bool):
    if gate.is_cuda and gate.numel() > 0:
        from ..engine import decoder

        with torch.cuda.device(gate.device):
            y, gate8, up8 = decoder.swiglu8_forward(gate, up, keep)
        return y, (*gate8, *up8) if keep else ()
    return (F.silu(gate.float()) * up.float()).to(gate.dtype), (*_host_pack(gate), *_host_pack(up)) if keep else ()


def _swiglu_backward(grad: Tensor, kept, with_y: bool):
    if grad.is_cuda and grad.numel() > 0:
        from ..engine import decoder

        with torch.cuda.device(grad.device):
            return decoder.swiglu8_backward(grad, decoder.Kept8(*kept[:2]), decoder.Kept8(*kept[2:]), with_y)
    dim = grad.shape[1]
    g, u = _host_unpack(kept[0], kept[1], dim, torch.float32), _host_unpack(kept[2], kept[3], dim, torch.float32)
    s, d = torch.sigmoid(g), grad.float()
    return ((d * u * s * (1.0 + g * (1.0 - s))).to(grad.dtype), (d * g * s).to(grad.dtype), (g * s * u).to(grad.dtype) if with_y else None)


class _SwiGLU8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up):
        y, kept = _swiglu_forward(gate, up, keep=True)
        ctx.save_for_backward(*kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return _swiglu_backward(grad, ctx.saved_tensors, with_y=False)[:2]


class _SwiGLULinear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, weight):
        y, kept = _swiglu_forward(gate, up, keep=True)
        ctx.save_for_backward(weight, *kept)
        return F.linear(y, weight)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        weight, *kept = ctx.saved_tensors
        want_weight = ctx.needs_input_grad[2]
        d_gate, d_up, y = _swiglu_backward(grad @ weight, kept, with_y=want_weight)
        return d_gate, d_up, grad.t() @ y if want_weight else None


def swiglu8(gate: Tensor, up: Tensor) -> Tensor:
    """``silu(gate) * up``; the backward pass works from both kept in 8 bits.  Differentiable once."""
    _check_swiglu(gate, up)
    flat = (gate.reshape(-1, gate.shape[-1]), up.reshape(-1, up.shape[-1]))
    if not torch.is_grad_enabled() or not (gate.requires_grad or up.requires_grad):
        return _swiglu_forward(*flat, keep=False)[0].view(gate.shape)
    return _SwiGLU8.apply(*flat).view(gate.shape)


def swiglu_linear8(gate: Tensor, up: Tensor, weight: Tensor) -> Tensor:
    """``(silu(gate) * up) @ weight.T``; only gate and up are kept, in 8 bits: 2 bytes and a bit of each pair of features instead of 6."""
    _check_swiglu(gate, up)
    if weight.ndim != 2 or weight.shape[1] != gate.shape[-1] or weight.dtype != gate.dtype or weight.device != gate.device:
        raise ValueError(f"weight must be (out, {gate.shape[-1]}) {gate.dtype} on {gate.device}, got {tuple(weight.shape)} {weight.dtype} on {weight.device}.")
    flat = (gate.reshape(-1, gate.shape[-1]), up.reshape(-1, up.shape[-1]))
    if not torch.is_grad_enabled() or not (gate.requires_grad or up.requires_grad or weight.requires_grad):
        out = F.linear(_swiglu_forward(*flat, keep=False)[0], weight)
    else:
        out = _SwiGLULinear8.apply(*flat, weight)
    return out.view(*gate.shape[:-1], weight.shape[0])


__all__ = ["Packed8", "checkpoint8", "pack8", "swiglu8", "swiglu_linear8", "unpack8"]

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

import functools
import math
from typing import Callable, Iterable, NamedTuple, Tuple

import torch
import torch.nn.functional as F
from torch import Tensor
from torch.autograd.function import once_differentiable

GROUP = 64
DTYPES = (torch.bfloat16, torch.float16, torch.float32)
SMALLEST_SCALE = 2.0 ** -126
LARGEST_SCALE = float.fromhex("0x1.020406p+121")      # 127 of it are a finite fp32 number


class Packed8(NamedTuple):
    """A tensor kept in 8 bits: what :func:`unpack8` needs."""

    values: Tensor            # int8 (rows, features rounded up to 8)
    scales: Tensor            # fp32 (rows, groups of 64 features)
    shape: torch.Size
    dtype: torch.dtype

    def bytes(self) -> int:
        return self.values.numel() + 4 * self.scales.numel()


@functools.cache
def _native():
    from ..engine import decoder

    return decoder.native


def _on_device(x: Tensor) -> bool:
    return x.is_cuda and x.numel() > 0


def _check_values(name: str, x: Tensor) -> None:
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name} must be (..., features), got {tuple(x.shape)}.")
    if x.dtype not in DTYPES:
        raise TypeError(f"{name} must be one of {DTYPES}, got {x.dtype}.")


def _host_pack(x: Tensor) -> Tuple[Tensor, Tensor]:
    rows, dim = x.shape
    groups = -(-dim // GROUP)
    v = F.pad(x.float(), (0, groups * GROUP - dim)).view(rows, groups, GROUP)
    scales = (v.abs().amax(dim=2) / 127.0).clamp(min=SMALLEST_SCALE, max=LARGEST_SCALE)
    scales = torch.where(torch.isfinite(v).all(dim=2), scales, torch.full_like(scales, float("nan")))
    values = torch.nan_to_num(torch.round(v / scales.unsqueeze(2)), nan=0.0).to(torch.int8).view(rows, groups * GROUP)
    return values[:, : -(-dim // 8) * 8].contiguous(), scales


def _host_unpack(values: Tensor, scales: Tensor, dim: int, dtype: torch.dtype) -> Tensor:
    return (values[:, :dim].float() * scales.repeat_interleave(GROUP, dim=1)[:, :dim]).to(dtype)


def pack8(x: Tensor) -> Packed8:
    """``x`` (..., features) in 8 bits; no gradients."""
    _check_values("x", x)
    if _on_device(x):
        values, scales = _native().pack8(x)
    else:
        values, scales = _host_pack(x.detach().reshape(-1, x.shape[-1]))
    return Packed8(values, scales, x.shape, x.dtype)


def unpack8(packed: Packed8) -> Tensor:
    """The values that ``packed`` stands for, in the dtype it was made from."""
    values, scales, shape, dtype = packed
    rows, dim = values.shape[0], shape[-1]
    if math.prod(shape) != rows * dim or values.shape != (rows, -(-dim // 8) * 8) or scales.shape != (rows, -(-dim // GROUP)):
        raise ValueError(f"values {tuple(values.shape)} and scales {tuple(scales.shape)} do not hold a tensor of shape {tuple(shape)}.")
    if values.dtype != torch.int8 or scales.dtype != torch.float32 or dtype not in DTYPES:
        raise TypeError(f"values are int8 and scales float32, got {values.dtype} and {scales.dtype} for {dtype}.")
    if values.device != scales.device:
        raise ValueError(f"values and scales must be on one device, got {values.device} and {scales.device}.")
    values, scales = values.contiguous(), scales.contiguous()
    if _on_device(values):
        return _native().unpack8(values, scales, shape, dtype)
    return _host_unpack(values, scales, dim, dtype).view(shape)


def _parameters_of(function: Callable) -> Iterable[Tensor]:
    """Those of a module, or of the module whose method it is."""
    while isinstance(function, functools.partial):
        function = function.func
    owner = function if isinstance(function, torch.nn.Module) else getattr(function, "__self__", None)
    return owner.parameters() if isinstance(owner, torch.nn.Module) else ()


def _holds_tensors(value) -> bool:
    """Whether ``value`` is a container with a tensor somewhere in it."""
    inside = value.values() if isinstance(value, dict) else value if isinstance(value, (tuple, list)) else ()
    return any(isinstance(v, Tensor) or _holds_tensors(v) for v in inside)


def _reaches_others(outputs: Iterable[Tensor], known: Iterable[Tensor]) -> bool:
    """Whether the graph behind ``outputs`` ends at a leaf that is not among ``known``."""
    known = {id(t) for t in known if isinstance(t, Tensor)}
    outputs = [o for o in outputs if isinstance(o, Tensor) and o.requires_grad]
    if any(o.grad_fn is None and id(o) not in known for o in outputs):
        return True
    nodes, seen = [o.grad_fn for o in outputs], set()
    while nodes:
        node = nodes.pop()
        if node is None or node in seen:
            continue
        seen.add(node)
        if node.name() == "torch::autograd::AccumulateGrad" and id(node.variable) not in known:
            return True
        nodes.extend(following for following, _ in node.next_functions)
    return False


class _Checkpoint8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, function, count, complete, x, *rest):
        ctx.function, ctx.count, ctx.complete = function, count, complete
        kind = x.device.type
        ctx.autocast = dict(device_type=kind, dtype=torch.get_autocast_dtype(kind), enabled=torch.is_autocast_enabled(kind),
                            cache_enabled=torch.is_autocast_cache_enabled())
        ctx.shape, ctx.dtype = x.shape, x.dtype
        packed = pack8(x)
        ctx.tensors = [isinstance(a, Tensor) for a in rest]
        ctx.plain = [None if t else a for a, t in zip(rest, ctx.tensors)]
        ctx.parameters = rest[count:]      # (themselves: hooks on saved tensors may bring back others; saved too, so that a change of theirs is noticed)
        ctx.save_for_backward(packed.values, packed.scales, *(a for a, t in zip(rest, ctx.tensors) if t))
        with torch.no_grad():
            outputs = function(x, *rest[:count])
        if not isinstance(outputs, (Tensor, tuple, list)) or not isinstance(outputs, Tensor) and any(map(_holds_tensors, outputs)):
            raise TypeError(f"checkpoint8: the function must return a tensor or a tuple of tensors, got {type(outputs).__name__} "
                            "or containers in it, whose tensors would have no gradients.")
        # what it returns without having made it (a parameter, a buffer) must not become an output of this node itself
        given = {id(a) for a in (x, *rest)}
        own = [o.detach() if isinstance(o, Tensor) and id(o) not in given else o for o in ([outputs] if isinstance(outputs, Tensor) else outputs)]
        return own[0] if isinstance(outputs, Tensor) else tuple(own)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        values, scales, *saved = ctx.saved_tensors
        x = unpack8(Packed8(values, scales, ctx.shape, ctx.dtype)).requires_grad_(ctx.needs_input_grad[3])
        saved = iter(saved)
        rest = [next(saved) if t else a for a, t in zip(ctx.plain, ctx.tensors)]
        # arguments become leaves of the second run; parameters are what the function holds itself
        arguments = [a.detach().requires_grad_(n) if isinstance(a, Tensor) else a
                     for a, n in zip(rest[: ctx.count], ctx.needs_input_grad[4:])]
        wanted = [a for a, n in zip([x, *arguments, *ctx.parameters], ctx.needs_input_grad[3:]) if n]
        with torch.enable_grad(), torch.autocast(**ctx.autocast):
            outputs = ctx.function(x, *arguments)
        outputs = (outputs,) if isinstance(outputs, Tensor) else tuple(outputs)
        if ctx.complete and _reaches_others(outputs, [x, *arguments, *ctx.parameters]):
            raise RuntimeError("checkpoint8: the function uses a tensor that requires gradients and is neither x, nor an argument, nor a parameter of the "
                               "module that the function is or belongs to; it would get none.  Hand it over as an argument, or say in "
                               "`parameters` which tensors get gradients.")
        pairs = [(o, g) for o, g in zip(outputs, grads) if isinstance(o, Tensor) and o.requires_grad and g is not None]
        found = iter(torch.autograd.grad([o for o, _ in pairs], wanted, [g for _, g in pairs], allow_unused=True) if pairs and wanted
                     else [None] * len(wanted))
        return (None, None, None, *(next(found) if n else None for n in ctx.needs_input_grad[3:]))


def checkpoint8(function: Callable, x: Tensor, *args, parameters: Iterable[Tensor] = None):
    """``function(x, *args)`` that keeps nothing but ``x`` in 8 bits (and ``args``, as they are) and is run again, from the kept ``x``, in
    the backward pass.

    ``function`` takes tensors or anything else, returns a tensor or a tuple of tensors, and does the same on every call (it must not
    draw random numbers); autocast is as it was in the first run.  Gradients reach ``x``, tensor ``args`` and ``parameters``: by default those of
    the module that ``function`` is, or that it is a method of, and then the backward pass is an error where the function uses any other tensor that requires
    gradients (of a closure, or inside another argument); ``parameters`` that are given are all that get gradients.  Without gradients of
    these it is a plain call.
    """
    _check_values("x", x)
    complete = parameters is None
    parameters = [p for p in (_parameters_of(function) if complete else parameters) if p.requires_grad]
    if not torch.is_grad_enabled() or not any(isinstance(a, Tensor) and a.requires_grad for a in (x, *args, *parameters)):
        return function(x, *args)
    return _Checkpoint8.apply(function, len(args), complete, x, *args, *parameters)


def _check_swiglu(gate: Tensor, up: Tensor) -> None:
    _check_values("gate", gate)
    if gate.shape != up.shape or gate.dtype != up.dtype or gate.device != up.device:
        raise ValueError(f"gate and up must match, got {tuple(gate.shape)} {gate.dtype} {gate.device} and {tuple(up.shape)} {up.dtype} {up.device}.")


def _host_swiglu(gate: Tensor, up: Tensor) -> Tensor:
    return (F.silu(gate.float()) * up.float()).to(gate.dtype)


def _host_swiglu_gradients(grad: Tensor, kept) -> Tuple[Tensor, Tensor, Tensor]:
    """Gradients of gate and up, and the activation, at the kept values."""
    dim = grad.shape[1]
    g, u = _host_unpack(kept[0], kept[1], dim, torch.float32), _host_unpack(kept[2], kept[3], dim, torch.float32)
    s, d = torch.sigmoid(g), grad.float()
    return (d * u * s * (1.0 + g * (1.0 - s))).to(grad.dtype), (d * g * s).to(grad.dtype), (g * s * u).to(grad.dtype)


class _SwiGLU8(torch.autograd.Function):
    """CPU tensors, and empty ones anywhere: with a weight, the linear layer behind it too."""

    @staticmethod
    def forward(ctx, gate, up, weight):
        ctx.save_for_backward(weight, *_host_pack(gate), *_host_pack(up))
        y = _host_swiglu(gate, up)
        with torch.autocast(gate.device.type, enabled=False):
            return y if weight is None else F.linear(y, weight)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        weight, *kept = ctx.saved_tensors
        with torch.autocast(grad.device.type, enabled=False):
            d_gate, d_up, y = _host_swiglu_gradients(grad if weight is None else grad @ weight, kept)
            return d_gate, d_up, grad.t() @ y if ctx.needs_input_grad[2] else None


def swiglu8(gate: Tensor, up: Tensor) -> Tensor:
    """``silu(gate) * up``; the backward pass works from both kept in 8 bits.  Differentiable once."""
    _check_swiglu(gate, up)
    if _on_device(gate):
        return _native().swiglu8(gate, up)
    dim = gate.shape[-1]
    return _SwiGLU8.apply(gate.reshape(-1, dim), up.reshape(-1, dim), None).view(gate.shape)


def swiglu_linear8(gate: Tensor, up: Tensor, weight: Tensor) -> Tensor:
    """``(silu(gate) * up) @ weight.T``; only gate and up are kept, in 8 bits: 2.1 bytes of each pair of features instead of the 8
    that eager torch keeps (gate, silu(gate), up and their product).
    In the type of its arguments, under autocast too."""
    _check_swiglu(gate, up)
    if weight.ndim != 2 or weight.shape[1] != gate.shape[-1] or weight.dtype != gate.dtype or weight.device != gate.device:
        raise ValueError(f"weight must be (out, {gate.shape[-1]}) {gate.dtype} on {gate.device}, got {tuple(weight.shape)} {weight.dtype} on {weight.device}.")
    if _on_device(gate):
        return _native().swiglu_linear8(gate, up, weight)
    dim = gate.shape[-1]
    return _SwiGLU8.apply(gate.reshape(-1, dim), up.reshape(-1, dim), weight).view(*gate.shape[:-1], weight.shape[0])


__all__ = ["Packed8", "checkpoint8", "pack8", "swiglu8", "swiglu_linear8", "unpack8"]

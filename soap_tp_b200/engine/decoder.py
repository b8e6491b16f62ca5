"""Device side of the operators of a decoder's training step (``csrc/cross_entropy.cu``, ``csrc/gemm16.cu``,
``csrc/residual_norm.cu``, ``csrc/activation8.cu``).

Everything runs on the current stream of the tensors' device with scratch from torch's allocator, which belongs to that stream (or to
the graph that is being captured), so calls on several streams and captured graphs share nothing.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch
from torch import Tensor

from . import kernels as k
from .kernels import _C

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
LOGIT_PART, SPLIT_COUNTERS, SPLIT_SCRATCH = _C.LOGIT_PART, _C.SPLIT_COUNTERS, _C.SPLIT_SCRATCH


def _rows16(x: Tensor) -> Tensor:
    """``x`` (rows, depth) as the tensor cores' loads take it: unit stride along depth, rows 16 bytes apart or a multiple of that.
    Anything else is copied once."""
    if x.stride(1) == 1 and x.stride(0) % 8 == 0 and x.stride(0) >= x.shape[1] and x.data_ptr() % 16 == 0:
        return x
    if x.shape[0] == 1 and x.stride(1) == 1 and x.data_ptr() % 16 == 0 and x.shape[1] % 8 == 0:
        return x.as_strided(x.shape, (x.shape[1], 1))
    padded = x.new_empty((x.shape[0], k.round_up(x.shape[1], 8)))[:, : x.shape[1]]
    padded.copy_(x)
    return padded


class Head:
    """One call's hidden states, this rank's words and the targets, ready for the kernels (``csrc/cross_entropy.h``)."""

    def __init__(self, hidden: Tensor, weight: Tensor, targets: Tensor, ignore_index: int, first_word: int, vocabulary: int) -> None:
        self.hidden, self.weight, self.targets = _rows16(hidden), _rows16(weight), targets.to(torch.int64).contiguous()
        self.tokens, self.depth, self.words = hidden.shape[0], hidden.shape[1], weight.shape[0]
        self.device, self.dtype = hidden.device, hidden.dtype
        # how many tokens count, which they are and their targets' columns; their hidden states, used unless all count
        self.numbers_of = torch.empty(1 + 2 * self.tokens + SPLIT_COUNTERS, dtype=torch.int32, device=self.device)
        self.packed = torch.empty((self.tokens, k.round_up(self.depth, 8)), dtype=self.dtype, device=self.device)
        self.problem = [self.hidden.data_ptr(), self.hidden.stride(0), self.weight.data_ptr(), self.weight.stride(0), self.tokens, self.depth,
                        self.words, int(self.dtype == torch.bfloat16), self.targets.data_ptr(), ignore_index, first_word, vocabulary,
                        self.numbers_of.data_ptr(), self.packed.data_ptr(), self.packed.shape[1]]
        self.status = k.status_word(self.device).data_ptr()

    def prepare(self, d_hidden: Optional[Tensor] = None) -> None:
        """Finds the tokens that count; the rows of ``d_hidden`` that belong to the others are cleared."""
        _C.head_prepare(self.problem, [0 if d_hidden is None else d_hidden.data_ptr(), self.depth, k._stream()])
        k._count("head_count_kernel")
        k._count("head_gather_kernel")

    def turns(self, workspace_bytes: int):
        """Tokens a turn, and the pitch of their logits in 16 bits: as many as the workspace holds, 256 at least."""
        pitch = k.round_up(self.words, 64)
        return min(self.tokens, max(256, workspace_bytes // (2 * pitch) // 256 * 256)), pitch

    def parts(self, rows: int) -> Tensor:
        return torch.empty((-(-self.words // LOGIT_PART), rows, 2), dtype=torch.float32, device=self.device)

    def statistics(self, first: int, rows: int, parts: Tensor, lse: Tensor, picked: Tensor, logits: Optional[Tensor] = None) -> None:
        """Log-sum-exp over this rank's words and the target's logit where this rank has it (0 elsewhere), of ``rows`` of the tokens
        that count; the exponentials stay in ``logits``."""
        _C.head_statistics(self.problem, [first, rows, 0 if logits is None else logits.data_ptr(), 0 if logits is None else logits.shape[1],
                                          parts.data_ptr(), lse.data_ptr(), picked.data_ptr(), self.status, k._stream()])
        k._count("gemm16_kernel")
        k._count("head_join_kernel")

    def loss(self, lse: Tensor, picked: Tensor, reduction: str) -> Tensor:
        loss = torch.empty(self.tokens if reduction == "none" else (), dtype=torch.float32, device=self.device)
        _C.head_losses(self.problem, [lse.data_ptr(), picked.data_ptr(), REDUCTIONS[reduction], loss.data_ptr(), k._stream()])
        k._count("head_losses_kernel")
        return loss


class HeadGradients:
    """Gradients of a head's hidden states and weight (those that are wanted), made turn by turn from the tokens' softmax."""

    def __init__(self, head: Head, want_hidden: bool, want_weight: bool, workspace_bytes: int) -> None:
        self.head = head
        self.rows, pitch = head.turns(workspace_bytes)
        device, dtype = head.device, head.dtype
        self.logits = torch.empty((self.rows, pitch), dtype=dtype, device=device)
        self.hidden = torch.empty((head.tokens, head.depth), dtype=dtype, device=device) if want_hidden else None
        self.weight = torch.empty((head.words, head.depth), dtype=dtype, device=device) if want_weight else None
        several = want_weight and self.rows < head.tokens
        self.sum = torch.empty((head.words, k.round_up(head.depth, 32)), dtype=torch.float32, device=device) if several else None
        self.factor = torch.empty(1 + head.tokens, dtype=torch.float32, device=device)      # alpha, then a factor for each token
        self.split_parts = torch.empty(SPLIT_SCRATCH, dtype=torch.float32, device=device)

    def turns(self):
        for first in range(0, self.head.tokens, self.rows):
            yield first, min(self.rows, self.head.tokens - first)

    def factors(self, reduction: str, grad_loss: Optional[Tensor]) -> None:
        alpha = self.factor.data_ptr()
        _C.head_factors(self.head.problem, [REDUCTIONS[reduction], 0 if grad_loss is None else grad_loss.data_ptr(), alpha + 4, alpha, k._stream()])
        k._count("head_factors_kernel")

    def add(self, first: int, rows: int, lse: Tensor, parts: Optional[Tensor] = None, picked: Optional[Tensor] = None) -> None:
        """One turn: from the exponentials that ``Head.statistics`` left in ``logits``, with their ``parts`` and ``picked``, or anew."""
        head, alpha = self.head, self.factor.data_ptr()
        _C.head_gradients(head.problem, [
            first, rows, self.logits.data_ptr(), self.logits.shape[1], 0 if parts is None else parts.data_ptr(), lse.data_ptr(),
            0 if picked is None else picked.data_ptr(), alpha + 4, alpha,
            0 if self.hidden is None else self.hidden.data_ptr(), head.depth, 0 if self.weight is None else self.weight.data_ptr(), head.depth,
            0 if self.sum is None else self.sum.data_ptr(), 0 if self.sum is None else self.sum.shape[1],
            self.split_parts.data_ptr(), head.status, k._stream()])
        k._count("head_rescale_kernel" if parts is not None else "gemm16_kernel")
        for wanted in (self.hidden, self.weight):
            if wanted is not None:
                k._count("gemm16_kernel")


def scale_gradients(factor: Tensor, a: Optional[Tensor], b: Optional[Tensor]) -> None:
    """Contiguous bf16 gradients times ``factor`` (one fp32 value), in place; nothing is moved where it is one."""
    _C.scale_gradients([factor.data_ptr(), 0 if a is None else a.data_ptr(), 0 if a is None else a.numel(),
                        0 if b is None else b.data_ptr(), 0 if b is None else b.numel(), k._stream()])
    k._count("scale_gradients_kernel")
    k.mark_written(a, b)


VALUE_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
SCALE_GROUP = _C.SCALE_GROUP


def _rows(x: Tensor) -> Tensor:
    """``x`` (rows, dim) with unit stride along the rows; anything else is copied."""
    return x if x.shape[1] == 1 or x.stride(1) == 1 else x.contiguous()


def _address(x: Optional[Tensor]) -> list:
    return [0, 0] if x is None else [x.data_ptr(), x.stride(0)]


def _pointer(x: Optional[Tensor]) -> int:
    return 0 if x is None else x.data_ptr()


class Kept8(NamedTuple):
    """Rows kept in 8 bits: whole numbers (rows, dim rounded up to 8) and a scale for every 64 of them."""

    values: Tensor
    scales: Tensor

    @staticmethod
    def empty(rows: int, dim: int, device: torch.device) -> "Kept8":
        return Kept8(torch.empty((rows, k.round_up(dim, 8)), dtype=torch.int8, device=device),
                     torch.empty((rows, -(-dim // SCALE_GROUP)), dtype=torch.float32, device=device))

    def numbers(self) -> list:
        return [self.values.data_ptr(), self.values.shape[1], self.scales.data_ptr()]


def pack8(x: Tensor) -> Kept8:
    x = _rows(x)
    kept = Kept8.empty(x.shape[0], x.shape[1], x.device)
    _C.pack8(VALUE_TYPES[x.dtype], [x.data_ptr(), x.stride(0), x.shape[0], x.shape[1], *kept.numbers(), k._stream()])
    k._count("pack8_kernel")
    return kept


def unpack8(kept: Kept8, dim: int, dtype: torch.dtype) -> Tensor:
    out = torch.empty((kept.values.shape[0], dim), dtype=dtype, device=kept.values.device)
    _C.unpack8(VALUE_TYPES[dtype], [*kept.numbers(), out.shape[0], dim, out.data_ptr(), dim, k._stream()])
    k._count("unpack8_kernel")
    return out


def swiglu8_forward(gate: Tensor, up: Tensor, keep: bool) -> Tuple[Tensor, Optional[Kept8], Optional[Kept8]]:
    gate, up = _rows(gate), _rows(up)
    rows, dim = gate.shape
    y = torch.empty((rows, dim), dtype=gate.dtype, device=gate.device)
    kept = (Kept8.empty(rows, dim, gate.device), Kept8.empty(rows, dim, gate.device)) if keep else (None, None)
    numbers = [*_address(gate), *_address(up), rows, dim, y.data_ptr(), dim, k._stream()]
    if keep:
        numbers += kept[0].numbers() + kept[1].numbers()
    _C.swiglu8_forward(VALUE_TYPES[gate.dtype], numbers)
    k._count("swiglu8_forward_kernel")
    return y, kept[0], kept[1]


def swiglu8_backward(grad: Tensor, gate8: Kept8, up8: Kept8, with_y: bool) -> Tuple[Tensor, Tensor, Optional[Tensor]]:
    """Gradients of gate and up, and with ``with_y`` the activation at the kept values."""
    grad = _rows(grad)
    rows, dim = grad.shape
    out = [torch.empty((rows, dim), dtype=grad.dtype, device=grad.device) for _ in range(2 + with_y)]
    _C.swiglu8_backward(VALUE_TYPES[grad.dtype], [*_address(grad), *gate8.numbers(), *up8.numbers(), rows, dim, out[0].data_ptr(),
                                                  out[1].data_ptr(), out[2].data_ptr() if with_y else 0, dim, k._stream()])
    k._count("swiglu8_backward_kernel")
    return out[0], out[1], out[2] if with_y else None


def _norm_numbers(x: Tensor, branch: Optional[Tensor], vectors, rms: Optional[Tensor], branch_rms: Optional[Tensor]) -> list:
    vector_type = next((v.dtype for v in vectors if v is not None), x.dtype)
    return [VALUE_TYPES[x.dtype], VALUE_TYPES[vector_type], x.shape[0], x.shape[1], *_address(x), *_address(branch),
            *(_pointer(v) for v in vectors), _pointer(rms), _pointer(branch_rms)]


def residual_norm_forward(x: Tensor, branch: Optional[Tensor], weight: Optional[Tensor], branch_weight: Optional[Tensor],
                          gate: Optional[Tensor], scale: float, eps: float):
    """``h`` (``x`` itself without a branch), ``y`` or None, and the reciprocal root mean squares of h and the branch."""
    x = _rows(x)
    branch = None if branch is None else _rows(branch)
    rows, dim = x.shape
    h = x if branch is None else torch.empty((rows, dim), dtype=x.dtype, device=x.device)
    y = None if weight is None else torch.empty((rows, dim), dtype=x.dtype, device=x.device)
    rms, branch_rms = torch.empty((2, rows), dtype=torch.float32, device=x.device)
    _C.residual_norm_forward(scale, eps, [*_norm_numbers(x, branch, (weight, branch_weight, gate), rms, branch_rms),
                                          0 if branch is None else h.data_ptr(), _pointer(y), dim, k._stream()])
    k._count("residual_norm_forward_kernel")
    return h, y, rms, branch_rms


def residual_norm_backward(h: Tensor, branch: Optional[Tensor], weight: Optional[Tensor], branch_weight: Optional[Tensor],
                           gate: Optional[Tensor], scale: float, eps: float, rms: Tensor, branch_rms: Tensor, grad_h: Optional[Tensor],
                           grad_y: Optional[Tensor], want):
    """Gradients of x, branch, weight, branch_weight and gate, those that ``want`` asks for (None elsewhere), each in memory of its own:
    where x and the branch are views of leaves, torch accumulates into what it is handed."""
    h = _rows(h)
    branch = None if branch is None else _rows(branch)
    grad_h = None if grad_h is None else _rows(grad_h)
    grad_y = None if grad_y is None else _rows(grad_y)
    rows, dim = h.shape
    d_x = torch.empty((rows, dim), dtype=h.dtype, device=h.device) if want[0] else None
    d_branch = torch.empty((rows, dim), dtype=h.dtype, device=h.device) if want[1] else None
    vectors = [torch.empty_like(v) if v is not None and w else None for v, w in zip((weight, branch_weight, gate), want[2:])]
    blocks = _C.residual_norm_blocks(rows, dim)
    partials = torch.empty((blocks, 3, dim), dtype=torch.float32, device=h.device) if any(v is not None for v in vectors) else None
    _C.residual_norm_backward(scale, eps, [
        *_norm_numbers(h, branch, (weight, branch_weight, gate), rms, branch_rms), *_address(grad_h), *_address(grad_y), _pointer(d_x),
        _pointer(d_branch), dim, _pointer(partials), blocks, *(_pointer(v) for v in vectors), k._stream()])
    k._count("residual_norm_backward_kernel")
    if partials is not None:
        k._count("norm_vectors_kernel")
    return (d_x, d_branch, *vectors)

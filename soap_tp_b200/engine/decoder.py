"""Device side of the operators of a decoder's training step: the native module ``soap_tp_b200._decoder`` (``csrc/decoder``).

Its operators are autograd functions in native code.  They run on the current stream of the tensors' device with scratch from torch's
allocator, which belongs to that stream (or to the graph that is being captured), so calls on several streams and captured graphs share nothing.
There is no eager-PyTorch fallback: a library that is missing is built in place, and if that fails the import error propagates.
"""
from __future__ import annotations

import torch

from . import kernels

try:
    from .. import _decoder as native  # type: ignore[attr-defined]
except ImportError:  # pragma: no cover - build on first use
    from .. import build_ext

    build_ext.build()
    from .. import _decoder as native  # type: ignore[attr-defined]

kernels.LAUNCHES_ELSEWHERE.append(native.launches)

REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_STATUS: dict = {}


def status(device: torch.device) -> int:
    """Address of the device's status word (``kernels.status_word``), which outlives the process's use of the device."""
    address = _STATUS.get(device)
    if address is None:
        address = _STATUS[device] = kernels.status_word(device).data_ptr()
    return address

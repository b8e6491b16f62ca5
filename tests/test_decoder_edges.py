"""Operators of a decoder's training step on CPU tensors, at the edges of what they accept: see also ``test_decoder_ops.py``."""
import pytest
import torch

from decoder_bounds import F32, half_step, within
from soap_tp_b200 import ops


# ---- the largest numbers ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_largest_values_stay_finite_in_eight_bits(dtype):
    x = torch.zeros(2, 130, dtype=dtype)
    x[0, 3], x[1, 70], x[1, 129] = torch.finfo(dtype).max, torch.finfo(dtype).min, torch.finfo(dtype).min
    back = ops.unpack8(ops.pack8(x))
    # the scale is rounded once or a step below that, the product once, the result once
    within(back, (x.double(), (half_step(dtype) + 4 * F32) * x.double().abs()))
    x[0, 5] = float("inf")
    assert bool(ops.unpack8(ops.pack8(x))[0, :64].isnan().all())

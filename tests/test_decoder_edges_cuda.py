"""Operators of a decoder's training step on the GPU, at the edges of what they accept: see also ``test_decoder_ops_cuda.py``."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from decoder_bounds import IGNORED, F32, half_step, head_exact, smallest, within
from test_decoder_ops_cuda import BF16, FP16, FP32, _check_head, _check_norm, _head, _no_timeouts, _rand  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- forward mode -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused(which, grad_mode):
    from soap_tp_b200 import ops

    plain = [_rand(4, 64, seed=i, dtype=BF16) for i in range(2)] + [_rand(8, 64, seed=2, dtype=BF16)]
    with torch.set_grad_enabled(grad_mode), forward_ad.dual_level():
        gate, up, weight = (forward_ad.make_dual(t, torch.ones_like(t)) if i == which else t for i, t in enumerate(plain))
        with pytest.raises(RuntimeError, match="jvp"):
            ops.swiglu_linear8(gate, up, weight)
        if which < 2:
            with pytest.raises(RuntimeError, match="jvp"):
                ops.swiglu8(gate, up)
            with pytest.raises(RuntimeError, match="jvp"):
                ops.residual_norm(gate, up, torch.ones(64, device="cuda"))
            with pytest.raises(RuntimeError, match="jvp"):
                ops.linear_cross_entropy(gate if which == 0 else up, weight, torch.zeros(4, dtype=torch.int64, device="cuda"))

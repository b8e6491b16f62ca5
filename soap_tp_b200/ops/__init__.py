"""Composable distributed operations of the tensor-parallel SOAP pipeline, and operators of a decoder's training step.

Thirteen public names are those of the reference's ``soap_tp.ops`` (``src/soap_tp/ops/__init__.py:23-37``) with the same
signatures.  The others serve the models that are trained (``models/llama_tp.py``): the head's cross entropy without logits
(``linear_cross_entropy``), norms fused with the residual stream (``residual_norm``, ``rms_norm``) and activations kept in 8 bits
(``checkpoint8``, ``swiglu8``, ``swiglu_linear8``, ``pack8``, ``unpack8``).
"""
from .activation8 import Packed8, checkpoint8, pack8, swiglu8, swiglu_linear8, unpack8
from ..layout import allocate_2d_block_cyclic
from .basis import (
    estimated_eigenvalue_order_2d_block_cyclic_,
    initialize_basis_2d_block_cyclic_,
    power_iteration_qr_2d_block_cyclic_,
    qr_2d_block_cyclic_,
    refresh_bases_and_transport_optimizer_state_,
)
from .elementwise import adam_update
from .gram import (
    update_left_preconditioner_2d_block_cyclic_,
    update_right_preconditioner_2d_block_cyclic_,
)
from .linear_cross_entropy import linear_cross_entropy
from .permute import permute_2d_block_cyclic_
from .redistribute import (
    redistribute_2d_block_cyclic_to_tp_shard,
    redistribute_tp_shard_to_2d_block_cyclic,
)
from .residual_norm import residual_norm, rms_norm
from .rotate import rotate_2d_block_cyclic_

__all__ = [
    "Packed8",
    "adam_update",
    "allocate_2d_block_cyclic",
    "checkpoint8",
    "estimated_eigenvalue_order_2d_block_cyclic_",
    "initialize_basis_2d_block_cyclic_",
    "linear_cross_entropy",
    "pack8",
    "permute_2d_block_cyclic_",
    "power_iteration_qr_2d_block_cyclic_",
    "qr_2d_block_cyclic_",
    "redistribute_2d_block_cyclic_to_tp_shard",
    "redistribute_tp_shard_to_2d_block_cyclic",
    "refresh_bases_and_transport_optimizer_state_",
    "residual_norm",
    "rms_norm",
    "rotate_2d_block_cyclic_",
    "swiglu8",
    "swiglu_linear8",
    "unpack8",
    "update_left_preconditioner_2d_block_cyclic_",
    "update_right_preconditioner_2d_block_cyclic_",
]

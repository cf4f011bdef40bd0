"""atex_b200: fused LayerNorm / InstanceNorm forward and gradient ops for NVIDIA
B200, exposing the public names of the reference package
(atex/nv_norms/__init__.py:6-13), and the norms of a transformer block beside them: RMS
normalisation and the gradients of the norms behind a residual add (rms_norm_ops.py), and the
per-head norm of queries and keys with rotary positions (rotary_ops.py).
"""
from .nv_norm_ops import (InstanceNormalization, InvalidArgumentError, LayerNormalization,
                          _instance_norm_grad, _layer_norm_grad, fused_instance_norm_grad_op,
                          fused_instance_norm_op, fused_layer_norm_grad_op, fused_layer_norm_op,
                          fused_layer_norm_residual_op, instance_norm, layer_norm)
from .rms_norm_ops import (RMSNormalization, fused_layer_norm_residual_grad_op, fused_rms_norm_grad_op,
                           fused_rms_norm_op, fused_rms_norm_residual_grad_op,
                           fused_rms_norm_residual_op, layer_norm_residual, rms_norm,
                           rms_norm_residual)
from .rotary_ops import (HeadNormRotary, fused_head_norm_rotary_grad_op, fused_head_norm_rotary_op,
                         head_norm_rotary, rotary_frequencies)

__all__ = [
    "fused_layer_norm_op", "fused_layer_norm_grad_op", "fused_instance_norm_op",
    "fused_instance_norm_grad_op", "_layer_norm_grad", "_instance_norm_grad",
    "LayerNormalization", "InstanceNormalization", "InvalidArgumentError", "layer_norm",
    "instance_norm", "fused_layer_norm_residual_op",
    "fused_rms_norm_op", "fused_rms_norm_grad_op", "fused_rms_norm_residual_op",
    "fused_rms_norm_residual_grad_op", "fused_layer_norm_residual_grad_op", "rms_norm",
    "rms_norm_residual", "layer_norm_residual", "RMSNormalization", "fused_head_norm_rotary_op",
    "fused_head_norm_rotary_grad_op", "head_norm_rotary", "rotary_frequencies", "HeadNormRotary",
]

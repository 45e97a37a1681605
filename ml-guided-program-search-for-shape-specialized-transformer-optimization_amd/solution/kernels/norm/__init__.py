"""gfx950 residual-plus-norm primitives and the norm of query and key heads."""

from .hip_qk_rotary import (
    HIP_QK_NORM_ROTARY_BACKEND,
    can_use_hip_qk_norm_rotary,
    hip_qk_norm_rotary,
    hip_qk_norm_rotary_available,
    rotary_table,
)
from .hip_residual import (
    HIP_LAYER_NORM_BACKEND,
    HIP_RESIDUAL_LAYER_NORM_BACKEND,
    HIP_RESIDUAL_RMS_NORM_BACKEND,
    HIP_RMS_NORM_BACKEND,
    can_use_hip_norm,
    can_use_hip_residual_norm,
    hip_layer_norm,
    hip_residual_layer_norm,
    hip_residual_norm_available,
    hip_residual_rms_norm,
    hip_rms_norm,
)

__all__ = [
    "HIP_LAYER_NORM_BACKEND",
    "HIP_QK_NORM_ROTARY_BACKEND",
    "HIP_RESIDUAL_LAYER_NORM_BACKEND",
    "HIP_RESIDUAL_RMS_NORM_BACKEND",
    "HIP_RMS_NORM_BACKEND",
    "can_use_hip_norm",
    "can_use_hip_qk_norm_rotary",
    "can_use_hip_residual_norm",
    "hip_layer_norm",
    "hip_qk_norm_rotary",
    "hip_qk_norm_rotary_available",
    "hip_residual_layer_norm",
    "hip_residual_norm_available",
    "hip_residual_rms_norm",
    "hip_rms_norm",
    "rotary_table",
]

"""gfx950 projection primitives."""

from .hip_linear_w4 import (
    HIP_LINEAR_W4_BACKEND,
    PackedLinearW4,
    can_use_hip_linear_w4,
    hip_linear_w4,
    hip_linear_w4_available,
    pack_linear_w4_codes,
    quantize_linear_w4,
)
from .hip_qkv_layout import (
    HIP_QKV_NATIVE_BHSD_BACKEND,
    VALUE_LAYOUTS,
    can_use_hip_qkv_native_bhsd,
    hip_qkv_native_bhsd,
    hip_qkv_native_bhsd_available,
    launch_config_is_valid,
    prevalidated_hip_qkv_native_bhsd,
    supported_shape,
)

__all__ = [
    "HIP_LINEAR_W4_BACKEND",
    "HIP_QKV_NATIVE_BHSD_BACKEND",
    "PackedLinearW4",
    "VALUE_LAYOUTS",
    "can_use_hip_linear_w4",
    "can_use_hip_qkv_native_bhsd",
    "hip_linear_w4",
    "hip_linear_w4_available",
    "hip_qkv_native_bhsd",
    "hip_qkv_native_bhsd_available",
    "launch_config_is_valid",
    "pack_linear_w4_codes",
    "prevalidated_hip_qkv_native_bhsd",
    "quantize_linear_w4",
    "supported_shape",
]

"""gfx950 choice of the tokens that a decoding step answers."""

from .hip_verify_draft import (
    HIP_VERIFY_DRAFT_BACKEND,
    can_use_hip_verify_draft,
    hip_verify_draft,
    hip_verify_draft_available,
)

__all__ = [
    "HIP_VERIFY_DRAFT_BACKEND",
    "can_use_hip_verify_draft",
    "hip_verify_draft",
    "hip_verify_draft_available",
]

"""gfx950 attention over a key/value cache (decoding)."""

from .hip_block_cache import (
    BLOCK_TOKENS,
    HIP_BLOCK_CACHE_APPEND_BACKEND,
    HIP_BLOCK_CACHE_ATTENTION_BACKEND,
    HIP_BLOCK_CACHE_READ_BACKEND,
    BlockCache,
    can_use_hip_block_cache_append,
    can_use_hip_block_cache_attention,
    can_use_hip_block_cache_read,
    hip_block_cache_append,
    hip_block_cache_attention,
    hip_block_cache_available,
    hip_block_cache_read,
)

__all__ = [
    "BLOCK_TOKENS",
    "BlockCache",
    "HIP_BLOCK_CACHE_APPEND_BACKEND",
    "HIP_BLOCK_CACHE_ATTENTION_BACKEND",
    "HIP_BLOCK_CACHE_READ_BACKEND",
    "can_use_hip_block_cache_append",
    "can_use_hip_block_cache_attention",
    "can_use_hip_block_cache_read",
    "hip_block_cache_append",
    "hip_block_cache_attention",
    "hip_block_cache_available",
    "hip_block_cache_read",
]

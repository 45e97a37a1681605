"""Norm of each query and key head with the position rotation, on gfx950.

No counterpart in the reference, whose attention takes the projected heads as
they are.  One pass over the packed projection's heads between the projection
and the attention, of whole sequences (solution/shape14/hip_streaming_dh64.py)
or over a cache (solution/kernels/attention/hip_block_cache.py): csrc/qk_rotary.hip.
"""

from __future__ import annotations

import torch

from ..hip._library import (
    SAH_NORM_LAYER,
    SAH_NORM_RMS,
    HipLibraryError,
    check_status,
    dtype_code,
    is_gfx950,
    launch_device,
    library_available,
    load_library,
    stream_handle,
)

HIP_QK_NORM_ROTARY_BACKEND = "hip_qk_norm_rotary"
SUPPORTED_HEAD_DIMS = frozenset({64, 128, 256})
SUPPORTED_DTYPES = frozenset({torch.bfloat16, torch.float16, torch.float32})
NORM_KINDS = {"layer": SAH_NORM_LAYER, "rms": SAH_NORM_RMS}


def rotary_table(
    positions: int,
    rotary_dim: int,
    *,
    base: float = 10000.0,
    device: torch.device | str = "cuda",
) -> torch.Tensor:
    """fp32 [positions, rotary_dim]: the cosines, then the sines, of position p
    times base ** (-2 i / rotary_dim), i < rotary_dim / 2.  Angles are formed in 64
    bits: in 32 the angle of position 1e5 would be off by 0.004."""

    if positions < 0 or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError("rotary_table needs positions >= 0 and an even rotary_dim")
    rates = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angles = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * rates
    return torch.cat([angles.cos(), angles.sin()], dim=1).float()


def hip_qk_norm_rotary_available() -> bool:
    """Whether the gfx950 library loads in this process."""

    return library_available()


def _heads_ok(value: torch.Tensor) -> bool:
    unit = 16 // value.element_size()
    strides = value.stride()
    if strides[3] != 1 or value.data_ptr() % 16 or (value.requires_grad and torch.is_grad_enabled()):
        return False
    return not any(stride % unit and size != 1 for size, stride in zip(value.shape[:3], strides))


def _param_dtype(parameters: tuple[torch.Tensor | None, ...], like: torch.Tensor) -> torch.dtype | None:
    """The one dtype of the parameters given (fp32 for none), or None where a
    parameter is not one the kernel reads."""

    found = None
    for parameter in parameters:
        if parameter is None:
            continue
        if (
            parameter.shape != like.shape[3:]
            or parameter.device != like.device
            or not parameter.is_contiguous()
            or parameter.data_ptr() % 16
            or (parameter.requires_grad and torch.is_grad_enabled())
            or parameter.dtype not in (torch.float32, like.dtype)
            or (found is not None and parameter.dtype is not found)
        ):
            return None
        found = parameter.dtype
    return torch.float32 if found is None else found


def can_use_hip_qk_norm_rotary(
    query: torch.Tensor,
    key: torch.Tensor,
    query_weight: torch.Tensor | None,
    key_weight: torch.Tensor | None,
    table: torch.Tensor | None,
    starts: torch.Tensor | None = None,
    *,
    query_bias: torch.Tensor | None = None,
    key_bias: torch.Tensor | None = None,
    eps: float = 1e-6,
    norm: str = "rms",
    interleaved: bool = False,
) -> bool:
    """Whether the kernel takes this request."""

    if query.ndim != 4 or key.ndim != 4 or query.dtype not in SUPPORTED_DTYPES or query.dtype is not key.dtype:
        return False
    batch, heads, seq_len, dim = query.shape
    if dim not in SUPPORTED_HEAD_DIMS or key.shape[0] != batch or key.shape[2:] != query.shape[2:]:
        return False
    if heads < 1 or key.shape[1] < 1 or query.device != key.device or batch * seq_len >= 2**31:
        return False
    if not (_heads_ok(query) and _heads_ok(key)) or norm not in NORM_KINDS or not eps >= 0:
        return False
    if _param_dtype((query_weight, query_bias, key_weight, key_bias), query) is None:
        return False
    if table is not None and (
        table.ndim != 2
        or table.dtype is not torch.float32
        or table.device != query.device
        or not table.is_contiguous()
        or table.data_ptr() % 16
        or not 0 < table.shape[1] <= dim
        or table.shape[1] % (8 if interleaved else 16)
        or table.requires_grad
    ):
        return False
    if starts is not None and (
        starts.dtype is not torch.int32
        or starts.shape != (batch,)
        or starts.device != query.device
        or not starts.is_contiguous()
    ):
        return False
    return is_gfx950(query.device) and library_available()


def hip_qk_norm_rotary(
    query: torch.Tensor,
    key: torch.Tensor,
    query_weight: torch.Tensor | None,
    key_weight: torch.Tensor | None,
    table: torch.Tensor | None,
    starts: torch.Tensor | None = None,
    *,
    query_bias: torch.Tensor | None = None,
    key_bias: torch.Tensor | None = None,
    eps: float = 1e-6,
    norm: str = "rms",
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor, str]:
    """Normalize every head of ``query`` [batch, heads, seq_len, head_dim] and
    ``key`` [batch, kv_heads, seq_len, head_dim] over its features ("rms" or
    "layer"), then rotate its first ``table.shape[1]`` features by the table row of
    the token's position ``starts[b] + i`` (``i`` without ``starts``).

    The inputs are views with any strides, head_dim contiguous (those of a packed
    projection); the outputs are new contiguous tensors, which the attentions read
    as given.  ``table`` is :func:`rotary_table`'s, or None for no rotation; pairs are
    features ``i`` and ``i + rotary_dim / 2``, or neighbours with ``interleaved``.
    Everything is formed in fp32 and rounded once.  A position outside the table
    makes NaN of the rotated features.
    """

    if not can_use_hip_qk_norm_rotary(
        query, key, query_weight, key_weight, table, starts,
        query_bias=query_bias, key_bias=key_bias, eps=eps, norm=norm, interleaved=interleaved,
    ):
        raise RuntimeError("HIP query/key norm with rotation is ineligible for the requested inputs")
    batch, heads, seq_len, dim = query.shape
    kv_heads = key.shape[1]
    query_out = torch.empty((batch, heads, seq_len, dim), dtype=query.dtype, device=query.device)
    key_out = torch.empty((batch, kv_heads, seq_len, dim), dtype=query.dtype, device=query.device)
    param_dtype = _param_dtype((query_weight, query_bias, key_weight, key_bias), query)
    pointers = [
        None if t is None else t.data_ptr()
        for t in (query, key, query_weight, query_bias, key_weight, key_bias, table, starts, query_out, key_out)
    ]
    try:
        with launch_device(query.device):
            status = load_library().sah_qk_norm_rotary(
                *pointers,
                batch,
                seq_len,
                heads,
                kv_heads,
                dim,
                *(0 if size == 1 else stride for size, stride in zip(query.shape[:3], query.stride())),
                *(0 if size == 1 else stride for size, stride in zip(key.shape[:3], key.stride())),
                0 if table is None else table.shape[1],
                0 if table is None else table.shape[0],
                int(interleaved),
                NORM_KINDS[norm],
                float(eps),
                dtype_code(query.dtype),
                dtype_code(param_dtype),
                stream_handle(query.device),
            )
            check_status(status, "sah_qk_norm_rotary")
    except HipLibraryError as exc:
        raise RuntimeError("HIP query/key norm with rotation execution failed") from exc
    return query_out, key_out, HIP_QK_NORM_ROTARY_BACKEND


__all__ = [
    "HIP_QK_NORM_ROTARY_BACKEND",
    "NORM_KINDS",
    "SUPPORTED_DTYPES",
    "SUPPORTED_HEAD_DIMS",
    "can_use_hip_qk_norm_rotary",
    "hip_qk_norm_rotary",
    "hip_qk_norm_rotary_available",
    "rotary_table",
]

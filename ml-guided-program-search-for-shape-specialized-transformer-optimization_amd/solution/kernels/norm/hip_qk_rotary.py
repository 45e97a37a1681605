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
    differentiated,
    dtype_code,
    launch,
    library_available,
    library_for,
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


def _strides(value: torch.Tensor, size: torch.Size, unit: int) -> tuple[int, int, int] | None:
    """Strides of the first three axes, 0 for an axis of size 1 (never stepped), or
    None for a tensor that the kernel does not read in place."""

    b, h, s, feature = value.stride()
    if size[0] == 1:
        b = 0
    if size[1] == 1:
        h = 0
    if size[2] == 1:
        s = 0
    if feature != 1 or b % unit or h % unit or s % unit or value.data_ptr() % 16:
        return None
    if differentiated(value):
        return None
    return b, h, s


def _param_dtype(
    parameters: tuple[torch.Tensor | None, ...], dim: int, index: int, like: torch.dtype
) -> torch.dtype | None:
    """The one dtype of the parameters given (fp32 for none), or None where a
    parameter is not one the kernel reads."""

    found = None
    for parameter in parameters:
        if parameter is None:
            continue
        dtype = parameter.dtype
        if (
            parameter.shape != (dim,)
            or parameter.get_device() != index
            or not parameter.is_contiguous()
            or parameter.data_ptr() % 16
            or differentiated(parameter)
            or (dtype is not torch.float32 and dtype is not like)
            or (found is not None and dtype is not found)
        ):
            return None
        found = dtype
    return torch.float32 if found is None else found


def _request(
    query: torch.Tensor,
    key: torch.Tensor,
    parameters: tuple[torch.Tensor | None, ...],
    table: torch.Tensor | None,
    starts: torch.Tensor | None,
    eps: float,
    norm: str,
    interleaved: bool,
) -> tuple | None:
    """The library, the device, the parameters' dtype and both strides of a request that
    the kernel takes, else None."""

    dtype, size, key_size, index = query.dtype, query.shape, key.shape, query.get_device()
    if dtype not in SUPPORTED_DTYPES or dtype is not key.dtype or len(size) != 4 or len(key_size) != 4:
        return None
    batch, heads, seq_len, dim = size
    if dim not in SUPPORTED_HEAD_DIMS or key_size[0] != batch or key_size[2] != seq_len or key_size[3] != dim:
        return None
    if heads < 1 or key_size[1] < 1 or index != key.get_device() or batch * seq_len >= 2**31:
        return None
    unit = 4 if dtype is torch.float32 else 8
    strides, key_strides = _strides(query, size, unit), _strides(key, key_size, unit)
    if strides is None or key_strides is None or norm not in NORM_KINDS or not eps >= 0:
        return None
    if table is not None:
        rows = table.shape
        if (
            len(rows) != 2
            or not 0 < rows[1] <= dim
            or rows[1] % (8 if interleaved else 16)
            or table.dtype is not torch.float32
            or table.get_device() != index
            or not table.is_contiguous()
            or table.data_ptr() % 16
            or table.requires_grad
            or differentiated(table)
        ):
            return None
    if starts is not None and (
        starts.dtype is not torch.int32
        or starts.shape != (batch,)
        or starts.get_device() != index
        or not starts.is_contiguous()
    ):
        return None
    param_dtype = _param_dtype(parameters, dim, index, dtype)
    library = library_for(index)
    return None if param_dtype is None or library is None else (library, index, param_dtype, strides, key_strides)


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

    parameters = (query_weight, query_bias, key_weight, key_bias)
    return _request(query, key, parameters, table, starts, eps, norm, interleaved) is not None


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

    parameters = (query_weight, query_bias, key_weight, key_bias)
    request = _request(query, key, parameters, table, starts, eps, norm, interleaved)
    if request is None:
        raise RuntimeError("HIP query/key norm with rotation is ineligible for the requested inputs")
    library, index, param_dtype, strides, key_strides = request
    batch, heads, seq_len, dim = query.shape
    rows, rotary_dim = (0, 0) if table is None else table.shape
    query_out = torch.empty_like(query, memory_format=torch.contiguous_format)
    key_out = torch.empty_like(key, memory_format=torch.contiguous_format)
    try:
        launch(
            index,
            library.sah_qk_norm_rotary,
            "sah_qk_norm_rotary",
            query.data_ptr(),
            key.data_ptr(),
            *[None if parameter is None else parameter.data_ptr() for parameter in parameters],
            None if table is None else table.data_ptr(),
            None if starts is None else starts.data_ptr(),
            query_out.data_ptr(),
            key_out.data_ptr(),
            batch,
            seq_len,
            heads,
            key.shape[1],
            dim,
            *strides,
            *key_strides,
            rotary_dim,
            rows,
            1 if interleaved else 0,
            NORM_KINDS[norm],
            float(eps),
            dtype_code(query.dtype),
            dtype_code(param_dtype),
        )
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

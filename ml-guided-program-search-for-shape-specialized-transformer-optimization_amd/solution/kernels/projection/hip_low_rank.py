"""Low-rank adapters of many requests beside a shared projection, on gfx950.

No counterpart in the reference.  The requests of a batch share a projection
(hip_linear_w4.py, solution/kernels/ffn/hip_linear_gelu.py), and each may have an adapter of
its own, two thin matrices whose product is added to the projection's weight; one call
adds them all to the projection's output (csrc/low_rank.hip)::

    packed, _ = hip_linear_w4(x, weight, bias)
    packed, _ = hip_low_rank_adapters(x, packed, adapters, indices, out=packed)
"""

from __future__ import annotations

from collections.abc import Sequence
from dataclasses import dataclass

import torch

from ..hip._library import (
    HipLibraryError,
    differentiated,
    dtype_code,
    launch,
    library_available,
    library_for,
)

HIP_LOW_RANK_ADAPTERS_BACKEND = "hip_low_rank_adapters"
SUPPORTED_DTYPES = frozenset({torch.bfloat16, torch.float16})
MAX_RANK = 128
_MAX_FEATURES = 2**24
_MAX_WORKGROUPS = (2**32 - 1) // 256  # of 16 tokens and 64 outputs each


@dataclass(frozen=True, eq=False)
class LowRankAdapters:
    """The adapters of one projection: adapter a adds ``scales[a] up[a] down[a]`` to its
    weight.

    ``down`` [adapters, rank, in_features] and ``up`` [adapters, out_features, rank] in
    bfloat16 or float16, rank a multiple of 8 up to 128, features multiples of 8 up to 2^24.
    ``scales`` [adapters] (float32, 1 without).  ``ranks`` [adapters] (int32) names each
    adapter's own rank where they differ; its directions from there to the next multiple
    of 8 are zeros, and those behind are not read.
    """

    down: torch.Tensor
    up: torch.Tensor
    scales: torch.Tensor | None = None
    ranks: torch.Tensor | None = None

    def __post_init__(self) -> None:
        down, up = self.down, self.up
        if down.ndim != 3 or up.ndim != 3 or down.dtype not in SUPPORTED_DTYPES or up.dtype != down.dtype:
            raise ValueError("down and up must be [adapters, rank, in] and [adapters, out, rank] in bfloat16 or float16")
        if up.shape[0] != down.shape[0] or up.shape[2] != down.shape[1]:
            raise ValueError("down and up do not belong together")
        if not 0 < self.rank <= MAX_RANK or self.rank % 8:
            raise ValueError("the rank must be a multiple of 8 up to 128")
        if not self.in_features or not self.out_features or self.in_features % 8 or self.out_features % 8:
            raise ValueError("in_features and out_features must be multiples of 8")
        if max(self.in_features, self.out_features) > _MAX_FEATURES:
            raise ValueError("in_features and out_features must be at most 2^24")
        for tensor, dtype in ((self.scales, torch.float32), (self.ranks, torch.int32)):
            if tensor is not None and (tensor.shape != (down.shape[0],) or tensor.dtype != dtype):
                raise ValueError("scales must be [adapters] in float32 and ranks [adapters] in int32")
        for tensor in (down, up, self.scales, self.ranks):
            if tensor is None:
                continue
            if not tensor.is_contiguous() or tensor.device != down.device or tensor.requires_grad or differentiated(tensor):
                raise ValueError("the adapters' tensors must be contiguous, on one device and need no gradient")
        if down.data_ptr() % 16 or up.data_ptr() % 16:
            raise ValueError("down and up must be 16-byte aligned")
        # tiles of 16 tokens that a launch takes (looked at on every call)
        object.__setattr__(self, "_most_tiles", _MAX_WORKGROUPS // -(-self.out_features // 64))

    @classmethod
    def pack(
        cls, adapters: Sequence[tuple[torch.Tensor, torch.Tensor, float]]
    ) -> "LowRankAdapters":
        """Lay out adapters ``(down [rank, in], up [out, rank], scale)`` of any ranks up
        to 128 once, filled up with zeros to a common one."""

        if not adapters:
            raise ValueError("there must be an adapter")
        first = adapters[0][0]
        for down, up, _ in adapters:
            if down.ndim != 2 or up.ndim != 2 or down.shape[0] != up.shape[1] or not 0 < down.shape[0] <= MAX_RANK:
                raise ValueError("an adapter is down [rank, in] and up [out, rank], of a rank up to 128")
            if down.shape[1] != first.shape[1] or up.shape[0] != adapters[0][1].shape[0]:
                raise ValueError("the adapters of a projection have its features")
            if any(t.dtype != first.dtype or t.device != first.device for t in (down, up)):
                raise ValueError("the adapters must have one type and device")
        rank = -(-max(down.shape[0] for down, _, _ in adapters) // 8) * 8
        packed_down = first.new_zeros((len(adapters), rank, first.shape[1]))
        packed_up = first.new_zeros((len(adapters), adapters[0][1].shape[0], rank))
        for place, (down, up, _) in enumerate(adapters):
            packed_down[place, : down.shape[0]] = down.detach()
            packed_up[place, :, : down.shape[0]] = up.detach()
        device = first.device
        return cls(
            packed_down.detach(),
            packed_up.detach(),
            torch.tensor([float(scale) for _, _, scale in adapters], dtype=torch.float32, device=device),
            torch.tensor([down.shape[0] for down, _, _ in adapters], dtype=torch.int32, device=device),
        )

    @property
    def rank(self) -> int:
        return self.down.shape[1]

    @property
    def in_features(self) -> int:
        return self.down.shape[2]

    @property
    def out_features(self) -> int:
        return self.up.shape[1]


def hip_low_rank_adapters_available() -> bool:
    """Whether the gfx950 library loads in this process."""

    return library_available()


def _strides(value: torch.Tensor) -> tuple[int, int] | None:
    """Strides of the sequences and tokens of [batch, seq, features] or [batch, features]
    (0 for an axis of size 1, never stepped), or None for rows that are not read in place."""

    size, strides = value.shape, value.stride()
    b = strides[0] if size[0] > 1 else 0
    s = strides[1] if len(size) == 3 and size[1] > 1 else 0
    if (size[-1] > 1 and strides[-1] != 1) or b % 8 or s % 8 or value.data_ptr() % 16:
        return None
    return b, s


def _span(value: torch.Tensor) -> tuple[int, int]:
    """The addresses that a tensor's elements lie between."""

    first = value.data_ptr()
    if not value.numel():
        return first, first
    last = sum((size - 1) * stride for size, stride in zip(value.shape, value.stride()))
    return first, first + (last + 1) * value.element_size()


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    (a0, a1), (b0, b1) = _span(a), _span(b)
    return a1 <= b0 or b1 <= a0


def _request(
    value: torch.Tensor,
    projected: torch.Tensor,
    adapters: LowRankAdapters,
    indices: torch.Tensor,
    counts: torch.Tensor | None,
) -> tuple | None:
    """The library, the device, batch, seq_len and the strides of value and projected of
    a request that the kernels take, else None."""

    down = adapters.down
    dtype, index, shape = down.dtype, down.get_device(), value.shape
    if value.dtype is not dtype or projected.dtype is not dtype or len(shape) not in (2, 3):
        return None
    if value.get_device() != index or projected.get_device() != index:
        return None
    if shape[-1] != down.shape[2] or projected.shape != (*shape[:-1], adapters.up.shape[1]):
        return None
    batch, seq_len = shape[0], shape[1] if len(shape) == 3 else 1
    if indices is None or batch * -(-seq_len // 16) > adapters._most_tiles:
        return None
    for words in (indices, counts):
        if words is not None and (
            words.dtype is not torch.int32
            or words.shape != (batch,)
            or not words.is_contiguous()
            or words.get_device() != index
        ):
            return None
    if differentiated(value) or differentiated(projected):
        return None
    value_strides, projected_strides = _strides(value), _strides(projected)
    if value_strides is None or projected_strides is None:
        return None
    library = library_for(index)
    return None if library is None else (library, index, batch, seq_len, value_strides, projected_strides)


def can_use_hip_low_rank_adapters(
    value: torch.Tensor,
    projected: torch.Tensor,
    adapters: LowRankAdapters,
    indices: torch.Tensor,
    counts: torch.Tensor | None = None,
) -> bool:
    """Whether the kernels take these tensors."""

    return _request(value, projected, adapters, indices, counts) is not None


def _check_out(
    out: torch.Tensor | None, value: torch.Tensor, projected: torch.Tensor, adapters: LowRankAdapters
) -> tuple[torch.Tensor, tuple[int, int]]:
    if out is None:
        shape = projected.shape
        return projected.new_empty(shape), ((shape[1] if len(shape) == 3 else 1) * shape[-1], shape[-1])
    strides = None
    if (
        out.dtype is projected.dtype
        and out.shape == projected.shape
        and out.get_device() == projected.get_device()
        and not differentiated(out)
    ):
        strides = _strides(out)
    same = out.data_ptr() == projected.data_ptr() and out.stride() == projected.stride()
    others = [value, adapters.down, adapters.up] + ([] if same else [projected])
    if strides is None or not all(_apart(out, other) for other in others):
        raise RuntimeError("HIP low-rank adapters output buffer does not match the request")
    return out, strides


def hip_low_rank_adapters(
    value: torch.Tensor,
    projected: torch.Tensor,
    adapters: LowRankAdapters,
    indices: torch.Tensor,
    counts: torch.Tensor | None = None,
    *,
    out: torch.Tensor | None = None,
) -> tuple[torch.Tensor, str]:
    """``projected + scale (value down^T) up^T`` with each sequence's own adapter.

    ``value`` is the projection's input [batch, seq_len, in_features], ``projected`` its
    output [batch, seq_len, out_features] (or both without the second axis, for one token a
    sequence; any strides of 8 elements' multiples, features contiguous).  Sequence b
    takes adapter ``indices[b]`` (int32); one outside [0, adapters) is none.  Rows from
    ``counts[b]`` on, and sequences without an adapter, are ``projected``'s as they are.
    fp32 accumulation, one rounding of the sum.  ``out`` receives the result: ``projected``
    itself, or a tensor apart from the inputs (by default a new one).
    """

    request = _request(value, projected, adapters, indices, counts)
    if request is None:
        raise RuntimeError("HIP low-rank adapters are ineligible for the requested inputs")
    library, index, batch, seq_len, value_strides, projected_strides = request
    output, output_strides = _check_out(out, value, projected, adapters)
    count, rank, in_features = adapters.down.shape
    out_features = adapters.up.shape[1]
    scales, ranks = adapters.scales, adapters.ranks
    try:
        size = library.sah_low_rank_adapters_workspace_bytes(batch, seq_len, in_features, out_features, rank)
        workspace = value.new_empty(size // 2) if size else None
        launch(
            index,
            library.sah_low_rank_adapters,
            "sah_low_rank_adapters",
            value.data_ptr(),
            projected.data_ptr(),
            adapters.down.data_ptr(),
            adapters.up.data_ptr(),
            None if scales is None else scales.data_ptr(),
            None if ranks is None else ranks.data_ptr(),
            indices.data_ptr(),
            None if counts is None else counts.data_ptr(),
            output.data_ptr(),
            batch,
            seq_len,
            in_features,
            out_features,
            count,
            rank,
            *value_strides,
            *projected_strides,
            *output_strides,
            dtype_code(value.dtype),
            None if workspace is None else workspace.data_ptr(),
            size,
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP low-rank adapters execution failed") from exc
    return output, HIP_LOW_RANK_ADAPTERS_BACKEND


__all__ = [
    "HIP_LOW_RANK_ADAPTERS_BACKEND",
    "LowRankAdapters",
    "MAX_RANK",
    "SUPPORTED_DTYPES",
    "can_use_hip_low_rank_adapters",
    "hip_low_rank_adapters",
    "hip_low_rank_adapters_available",
]

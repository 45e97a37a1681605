"""Linear layers with 4-bit weights for few rows, on gfx950.

No counterpart in the reference.  The projections of a decoding step, whose time
is the reading of the weights: codes of 4 bits (-7 to 7) and one scale for each
group of 32, 64 or 128 inputs of an output (csrc/linear_w4.hip).  Beside the
16-bit projections (solution/kernels/ffn/hip_linear_gelu.py), which are the
faster ones for many rows.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from ..hip._library import (
    SAH_ACTIVATION_GELU_EXACT,
    SAH_ACTIVATION_NONE,
    HipLibraryError,
    differentiated,
    dtype_code,
    launch,
    library_available,
    library_for,
)

HIP_LINEAR_W4_BACKEND = "hip_linear_w4"
SUPPORTED_GROUP_SIZES = frozenset({32, 64, 128})
SUPPORTED_DTYPES = frozenset({torch.bfloat16, torch.float16})
ACTIVATIONS = {"none": SAH_ACTIVATION_NONE, "gelu": SAH_ACTIVATION_GELU_EXACT}
_TILE_IN = 128
_MAX_ROW_STRIDE = 2**25
_TILE_OUT = 16
_LARGEST_CODE = 7


@dataclass(frozen=True, eq=False)
class PackedLinearW4:
    """A weight [out_features, in_features] in 4 bits, laid out once.

    ``codes``: int32 words [out_features / 16, in_features / 128, 64, 4], eight
    codes each, in the order that include/shape_aware_hip.h gives (a lane's four
    operands side by side).  ``scales``: [in_features / group_size, out_features] in
    the type of the inputs that it multiplies.
    """

    codes: torch.Tensor
    scales: torch.Tensor

    def __post_init__(self) -> None:
        codes, scales = self.codes, self.scales
        if codes.ndim != 4 or codes.shape[2:] != (64, 4) or codes.dtype != torch.int32 or not codes.numel():
            raise ValueError("codes must be int32 words [out / 16, in / 128, 64, 4]")
        if scales.ndim != 2 or scales.dtype not in SUPPORTED_DTYPES or scales.shape[1] != self.out_features:
            raise ValueError("scales must be [in / group_size, out] in bfloat16 or float16")
        if not scales.shape[0] or self.in_features % scales.shape[0] or self.group_size not in SUPPORTED_GROUP_SIZES:
            raise ValueError("the group size must be 32, 64 or 128")
        for tensor in (codes, scales):
            if not tensor.is_contiguous() or tensor.device != codes.device or tensor.requires_grad or differentiated(tensor):
                raise ValueError("codes and scales must be contiguous, on one device and need no gradient")
            if tensor.data_ptr() % 16:
                raise ValueError("codes and scales must be 16-byte aligned")

    @property
    def out_features(self) -> int:
        return self.codes.shape[0] * _TILE_OUT

    @property
    def in_features(self) -> int:
        return self.codes.shape[1] * _TILE_IN

    @property
    def group_size(self) -> int:
        return self.in_features // self.scales.shape[0]

    def dequantize(self) -> torch.Tensor:
        """The weight [out_features, in_features] in fp32."""

        bit = torch.arange(8, device=self.codes.device)
        low = 8 * (bit % 4) + 4 * (bit // 4)
        words = self.codes.long()[..., None]
        codes = ((words >> low) & 7) * (1 - 2 * ((words >> ((low + 7) % 32)) & 1))
        tiles_n, tiles_k = self.codes.shape[:2]
        codes = codes.reshape(tiles_n, tiles_k, 4, 16, 4, 8).permute(0, 3, 1, 4, 2, 5)
        codes = codes.reshape(self.out_features, -1, self.group_size)
        return (codes.float() * self.scales.t().float()[..., None]).reshape(self.out_features, self.in_features)


def pack_linear_w4_codes(codes: torch.Tensor, scales: torch.Tensor) -> PackedLinearW4:
    """Pack whole-number ``codes`` [out_features, in_features] in -7 .. 7 with
    ``scales`` [out_features, in_features / group_size] (bfloat16 or float16)."""

    if codes.ndim != 2 or scales.ndim != 2 or codes.is_floating_point() or codes.dtype == torch.bool:
        raise ValueError("codes and scales must be matrices, codes of whole numbers")
    out_features, in_features = codes.shape
    if not codes.numel() or out_features % _TILE_OUT or in_features % _TILE_IN:
        raise ValueError("out_features must be a multiple of 16 and in_features of 128")
    codes = codes.long()
    if int(codes.abs().max()) > _LARGEST_CODE:
        raise ValueError("codes must lie in -7 .. 7")
    if scales.shape[0] != out_features:
        raise ValueError("scales must have a row for each output")
    bit = torch.arange(8, device=codes.device)
    low = 8 * (bit % 4) + 4 * (bit // 4)
    # [out tile, lane % 16, in tile, step, lane / 16, element] -> [out tile, in tile, lane / 16, lane % 16, step, element]
    tiles = codes.reshape(out_features // 16, 16, in_features // 128, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)
    words = ((tiles.abs() << low) | ((tiles < 0).long() << ((low + 7) % 32))).sum(-1)
    words = torch.where(words >= 2**31, words - 2**32, words)
    words = words.to(torch.int32).reshape(out_features // 16, in_features // 128, 64, 4)
    return PackedLinearW4(words.contiguous(), scales.t().contiguous())


def quantize_linear_w4(weight: torch.Tensor, group_size: int = 128) -> PackedLinearW4:
    """Round ``weight`` [out_features, in_features] (bfloat16 or float16) to 4-bit
    codes with one scale a group, its largest magnitude over 7."""

    if weight.ndim != 2 or weight.dtype not in SUPPORTED_DTYPES:
        raise ValueError("weight must be a bfloat16 or float16 matrix")
    if group_size not in SUPPORTED_GROUP_SIZES or weight.shape[1] % group_size:
        raise ValueError("the group size must be 32, 64 or 128 and divide in_features")
    if not bool(torch.isfinite(weight).all()):
        raise ValueError("weight must be finite")
    groups = weight.detach().float().reshape(weight.shape[0], -1, group_size)
    scales = (groups.abs().amax(-1) / _LARGEST_CODE).to(weight.dtype)
    # codes for the scale as it is stored; a group of zeros keeps scale 0
    divisor = torch.where(scales > 0, scales.float(), torch.ones_like(scales, dtype=torch.float32))
    codes = torch.round(groups / divisor[..., None]).clamp_(-_LARGEST_CODE, _LARGEST_CODE)
    return pack_linear_w4_codes(codes.to(torch.int8).reshape(weight.shape), scales)


def hip_linear_w4_available() -> bool:
    """Whether the gfx950 library loads in this process."""

    return library_available()


def can_use_hip_linear_w4(
    value: torch.Tensor,
    weight: PackedLinearW4,
    bias: torch.Tensor | None = None,
    *,
    activation: str = "none",
) -> bool:
    """Whether the kernel takes this request."""

    return _request(value, weight, bias, activation) is not None


def _request(
    value: torch.Tensor, weight: PackedLinearW4, bias: torch.Tensor | None, activation: str
) -> tuple | None:
    """The library, the device, in_features, out_features, group size and row stride of
    a request that the kernel takes, else None."""

    scales = weight.scales
    dtype, index, shape = scales.dtype, scales.get_device(), value.shape
    groups, out_features = scales.shape
    in_features = weight.in_features
    if value.dtype is not dtype or value.get_device() != index or not shape or shape[-1] != in_features:
        return None
    if activation not in ACTIVATIONS or value.data_ptr() % 16:
        return None
    if differentiated(value):
        return None
    stride = _row_stride(shape, value.stride())
    if stride is None:
        return None
    if bias is not None and (
        bias.shape != (out_features,)
        or bias.dtype is not dtype
        or bias.get_device() != index
        or not bias.is_contiguous()
        or bias.data_ptr() % 8
        or differentiated(bias)
    ):
        return None
    library = library_for(index)
    return None if library is None else (library, index, in_features, out_features, in_features // groups, stride)


def _row_stride(shape: tuple[int, ...], strides: tuple[int, ...]) -> int | None:
    """The stride of a tensor's rows, taken as one axis; None where they are not
    at one stride that the kernel reads."""

    if 0 in shape:  # no rows
        return shape[-1]
    if strides[-1] != 1:
        return None
    stride, span = shape[-1], None
    for axis in range(len(shape) - 2, -1, -1):
        size, step = shape[axis], strides[axis]
        if size == 1:
            continue
        if span is None:
            stride = step
        elif step != span:
            return None
        span = step * size
    return stride if stride % 8 == 0 and 0 <= stride <= _MAX_ROW_STRIDE else None


def hip_linear_w4(
    value: torch.Tensor,
    weight: PackedLinearW4,
    bias: torch.Tensor | None = None,
    *,
    activation: str = "none",
) -> tuple[torch.Tensor, str]:
    """``act(value W^T + bias)`` of ``value`` [..., in_features], with W the codes
    times their groups' scales, fp32 accumulation and one rounding.  ``activation``
    is "none" or "gelu" (exact).  Any number of rows is right; it is meant for up to
    a few dozen."""

    request = _request(value, weight, bias, activation)
    if request is None:
        raise RuntimeError("HIP 4-bit linear is ineligible for the requested inputs")
    library, index, in_features, out_features, group_size, stride = request
    output = value.new_empty((*value.shape[:-1], out_features))
    try:
        launch(
            index,
            library.sah_linear_w4,
            "sah_linear_w4",
            value.data_ptr(),
            weight.codes.data_ptr(),
            weight.scales.data_ptr(),
            None if bias is None else bias.data_ptr(),
            output.data_ptr(),
            value.numel() // in_features,
            in_features,
            out_features,
            group_size,
            stride,
            out_features,
            dtype_code(value.dtype),
            ACTIVATIONS[activation],
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP 4-bit linear execution failed") from exc
    return output, HIP_LINEAR_W4_BACKEND


__all__ = [
    "ACTIVATIONS",
    "HIP_LINEAR_W4_BACKEND",
    "PackedLinearW4",
    "SUPPORTED_DTYPES",
    "SUPPORTED_GROUP_SIZES",
    "can_use_hip_linear_w4",
    "hip_linear_w4",
    "hip_linear_w4_available",
    "pack_linear_w4_codes",
    "quantize_linear_w4",
]

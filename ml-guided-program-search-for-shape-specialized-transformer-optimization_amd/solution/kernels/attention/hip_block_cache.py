"""Key/value cache in 8 bits and the attention that reads it, on gfx950.

No counterpart in the reference, whose forward takes whole sequences.  These
are the operators of a decoding step beside the causal attention of whole
sequences (solution/shape14/hip_streaming_dh64.py), in the manner of its
modules: ``can_use_*``, strict calls that return ``(..., marker)``, RuntimeError
"... ineligible ..." for inputs that the kernels do not take.

A step of one layer, for ``batch`` sequences of which ``starts`` tokens are held::

    query, key, _ = hip_qk_norm_rotary(query, key, wq, wk, table, starts)
    hip_block_cache_append(cache, key, value, starts)
    context, _ = hip_block_cache_attention(query, cache, starts)

and after the step's last layer ``starts += 1`` (or ``+= counts``).

:class:`BlockCache` describes the format; include/shape_aware_hip.h defines it.
"""

from __future__ import annotations

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

HIP_BLOCK_CACHE_APPEND_BACKEND = "hip_block_cache_append"
HIP_BLOCK_CACHE_READ_BACKEND = "hip_block_cache_read"
HIP_BLOCK_CACHE_ATTENTION_BACKEND = "hip_block_cache_attention"

BLOCK_TOKENS = 64
SUPPORTED_HEAD_DIMS = frozenset({64, 128})
SUPPORTED_DTYPES = frozenset({torch.bfloat16, torch.float16})
_MAX_LENGTH = 2**31 - 1
_MAX_SCALE = 2.0**127  # times log2(e) still in fp32's range


@dataclass(frozen=True, eq=False)
class BlockCache:
    """One layer's keys and values, in blocks of 64 tokens.

    ``block_table`` [batch, max_blocks] (int32) names the place of each block of
    a sequence among ``num_blocks``; layers that share their sequences' layout may
    share it.  A complete block holds e4m3 codes (bytes) and one power-of-two scale
    a head: ``key_codes`` [num_blocks, kv_heads, 64, head_dim] and ``key_scales``
    [num_blocks, kv_heads]; values feature by feature, ``value_codes`` [num_blocks,
    kv_heads, head_dim, 64].  The block that a sequence has not filled stands in 16
    bits in ``key_tail`` [batch, kv_heads, 64, head_dim] and ``value_tail`` [batch,
    kv_heads, head_dim, 64].
    """

    key_codes: torch.Tensor
    value_codes: torch.Tensor
    key_scales: torch.Tensor
    value_scales: torch.Tensor
    key_tail: torch.Tensor
    value_tail: torch.Tensor
    block_table: torch.Tensor

    def __post_init__(self) -> None:
        tail = self.key_tail
        if tail.ndim != 4 or tail.shape[2] != BLOCK_TOKENS or tail.shape[3] not in SUPPORTED_HEAD_DIMS:
            raise ValueError("key_tail must be [batch, kv_heads, 64, head_dim] with head_dim 64 or 128")
        if tail.dtype not in SUPPORTED_DTYPES:
            raise ValueError("the cache's tails must be bfloat16 or float16")
        batch, heads, _, dim = tail.shape
        if self.key_codes.ndim != 4 or self.block_table.ndim != 2 or heads < 1:
            raise ValueError("the cache's tensors do not belong together")
        blocks = self.key_codes.shape[0]
        expected = (
            (self.key_codes, (blocks, heads, BLOCK_TOKENS, dim), torch.uint8),
            (self.value_codes, (blocks, heads, dim, BLOCK_TOKENS), torch.uint8),
            (self.key_scales, (blocks, heads), torch.float32),
            (self.value_scales, (blocks, heads), torch.float32),
            (self.key_tail, (batch, heads, BLOCK_TOKENS, dim), tail.dtype),
            (self.value_tail, (batch, heads, dim, BLOCK_TOKENS), tail.dtype),
            (self.block_table, (batch, self.block_table.shape[1]), torch.int32),
        )
        for tensor, shape, dtype in expected:
            if tuple(tensor.shape) != shape or tensor.dtype != dtype:
                raise ValueError(f"the cache's tensors do not belong together: expected {dtype} {shape}")
            if not tensor.is_contiguous() or tensor.device != tail.device or tensor.requires_grad or differentiated(tensor):
                raise ValueError("the cache's tensors must be contiguous, on one device and need no gradient")
        for tensor in (self.key_codes, self.value_codes, self.key_tail, self.value_tail):
            if tensor.data_ptr() % 16:
                raise ValueError("the cache's codes and tails must be 16-byte aligned")
        # whether csrc/block_pool.hip's kernels take its sizes (looked at on every call):
        # copies and forks of blocks, and tokens taken back
        moves = heads <= 65536 and blocks <= _MAX_LENGTH
        goes_back = self.block_table.shape[1] <= _MAX_LENGTH // BLOCK_TOKENS and batch <= (2**32 - 1) // 256 // (2 * heads)
        object.__setattr__(self, "_moves", moves)
        object.__setattr__(self, "_goes_back", moves and goes_back)

    @classmethod
    def allocate(
        cls,
        batch: int,
        kv_heads: int,
        head_dim: int,
        *,
        max_tokens: int,
        num_blocks: int | None = None,
        dtype: torch.dtype = torch.bfloat16,
        device: torch.device | str = "cuda",
        block_table: torch.Tensor | None = None,
    ) -> "BlockCache":
        """An empty cache for sequences of up to ``max_tokens``.  By default every
        sequence has places of its own for all of them; with ``num_blocks`` given
        and no ``block_table``, no place is named yet (-1)."""

        width = max_tokens // BLOCK_TOKENS
        if block_table is not None:
            width = block_table.shape[1]
        if num_blocks is None:
            num_blocks = batch * width
            if block_table is None:
                block_table = torch.arange(num_blocks, dtype=torch.int32, device=device).reshape(batch, width)
        elif block_table is None:
            block_table = torch.full((batch, width), -1, dtype=torch.int32, device=device)
        codes = (num_blocks, kv_heads, BLOCK_TOKENS * head_dim)
        return cls(
            torch.zeros(codes, dtype=torch.uint8, device=device).view(num_blocks, kv_heads, BLOCK_TOKENS, head_dim),
            torch.zeros(codes, dtype=torch.uint8, device=device).view(num_blocks, kv_heads, head_dim, BLOCK_TOKENS),
            torch.ones((num_blocks, kv_heads), device=device),
            torch.ones((num_blocks, kv_heads), device=device),
            torch.zeros((batch, kv_heads, BLOCK_TOKENS, head_dim), dtype=dtype, device=device),
            torch.zeros((batch, kv_heads, head_dim, BLOCK_TOKENS), dtype=dtype, device=device),
            block_table,
        )

    @property
    def batch(self) -> int:
        return self.key_tail.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.key_tail.shape[1]

    @property
    def head_dim(self) -> int:
        return self.key_tail.shape[3]

    @property
    def max_tokens(self) -> int:
        """The most tokens that a sequence can hold: its table's blocks and a tail."""

        return min(self.block_table.shape[1] * BLOCK_TOKENS + BLOCK_TOKENS - 1, _MAX_LENGTH)

    def _pointers(self) -> tuple[int, ...]:
        return (
            self.key_codes.data_ptr(),
            self.value_codes.data_ptr(),
            self.key_scales.data_ptr(),
            self.value_scales.data_ptr(),
            self.key_tail.data_ptr(),
            self.value_tail.data_ptr(),
            self.block_table.data_ptr(),
        )


def hip_block_cache_available() -> bool:
    """Whether the gfx950 library loads in this process."""

    return library_available()


def _lengths_ok(lengths: torch.Tensor | None, batch: int, index: int) -> bool:
    return lengths is None or (
        lengths.dtype is torch.int32
        and lengths.shape == (batch,)
        and lengths.is_contiguous()
        and lengths.get_device() == index
    )


def _strides(value: torch.Tensor, size: torch.Size) -> tuple[int, int, int] | None:
    """Strides of the first three axes, 0 for an axis of size 1 (never stepped), or
    None for a tensor that the kernels do not read in place."""

    b, h, s, feature = value.stride()
    if size[0] == 1:
        b = 0
    if size[1] == 1:
        h = 0
    if size[2] == 1:
        s = 0
    if feature != 1 or b % 8 or h % 8 or s % 8 or value.data_ptr() % 16:
        return None
    if differentiated(value):
        return None
    return b, h, s


def _append_request(
    cache: BlockCache,
    key: torch.Tensor,
    value: torch.Tensor,
    starts: torch.Tensor,
    counts: torch.Tensor | None,
) -> tuple | None:
    """The library, the device and the strides of key and value where the append kernel
    takes the request, else None."""

    tail, size = cache.key_tail, key.shape
    dtype, index = tail.dtype, tail.get_device()
    if key.dtype is not dtype or value.dtype is not dtype or len(size) != 4 or value.shape != size:
        return None
    batch, heads, _, dim = tail.shape
    if size[0] != batch or size[1] != heads or size[3] != dim:
        return None
    if key.get_device() != index or value.get_device() != index:
        return None
    key_strides, value_strides = _strides(key, size), _strides(value, size)
    if key_strides is None or value_strides is None or starts is None:
        return None
    if not (_lengths_ok(starts, batch, index) and _lengths_ok(counts, batch, index)):
        return None
    library = library_for(index)
    return None if library is None else (library, index, key_strides, value_strides)


def can_use_hip_block_cache_append(
    cache: BlockCache,
    key: torch.Tensor,
    value: torch.Tensor,
    starts: torch.Tensor,
    counts: torch.Tensor | None = None,
) -> bool:
    """Whether the append kernel takes these tensors."""

    return _append_request(cache, key, value, starts, counts) is not None


def hip_block_cache_append(
    cache: BlockCache,
    key: torch.Tensor,
    value: torch.Tensor,
    starts: torch.Tensor,
    counts: torch.Tensor | None = None,
) -> str:
    """Append each sequence's new tokens to the cache, in place.

    ``key`` and ``value`` are [batch, kv_heads, seq_len, head_dim] (any strides,
    head_dim contiguous); sequence b holds ``starts[b]`` tokens and takes the first
    ``counts[b]`` rows, or all ``seq_len`` without ``counts``.  A block is coded when
    its 64th token comes, at a place that no other sequence of the call completes
    one at.  Blocks without a place in the cache are dropped, and the attention that
    would read them answers NaN.  A token with a non-finite key or value makes NaN of
    every query that attends to it, and of no other.

    Tokens are taken back by lowering ``starts``: within the sequence's incomplete
    block, or to a multiple of 64.  Not elsewhere below that block, whose tokens stand
    where the earlier block's stood before it was coded: to go back there, call
    :func:`hip_block_cache_take_back` first (or read the block's first tokens with
    :func:`hip_block_cache_read` and append them anew, from the multiple of 64 on).
    """

    request = _append_request(cache, key, value, starts, counts)
    if request is None:
        raise RuntimeError("HIP block cache append is ineligible for the requested inputs")
    library, index, key_strides, value_strides = request
    batch, heads, seq_len, dim = key.shape
    try:
        launch(
            index,
            library.sah_block_cache_append,
            "sah_block_cache_append",
            key.data_ptr(),
            value.data_ptr(),
            *cache._pointers(),
            starts.data_ptr(),
            None if counts is None else counts.data_ptr(),
            batch,
            heads,
            seq_len,
            dim,
            *key_strides,
            *value_strides,
            cache.key_codes.shape[0],
            cache.block_table.shape[1],
            dtype_code(key.dtype),
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP block cache append execution failed") from exc
    return HIP_BLOCK_CACHE_APPEND_BACKEND


def can_use_hip_block_cache_read(
    cache: BlockCache, firsts: torch.Tensor, lengths: torch.Tensor, tokens: int
) -> bool:
    """Whether the read kernel takes these tensors."""

    tail = cache.key_tail
    batch, index = tail.shape[0], tail.get_device()
    return (
        isinstance(tokens, int)
        and not isinstance(tokens, bool)
        and tokens >= 0
        and firsts is not None
        and lengths is not None
        and _lengths_ok(firsts, batch, index)
        and _lengths_ok(lengths, batch, index)
        and library_for(index) is not None
    )


def hip_block_cache_read(
    cache: BlockCache, firsts: torch.Tensor, lengths: torch.Tensor, tokens: int
) -> tuple[torch.Tensor, torch.Tensor, str]:
    """What the cache holds, in its 16-bit type: keys and values [batch, kv_heads,
    tokens, head_dim] of positions ``firsts[b] ..``, zeros before position 0 and from
    ``lengths[b]`` (the tokens that sequence b holds) on."""

    if not can_use_hip_block_cache_read(cache, firsts, lengths, tokens):
        raise RuntimeError("HIP block cache read is ineligible for the requested inputs")
    tail = cache.key_tail
    batch, heads, _, dim = tail.shape
    index = tail.get_device()
    key = tail.new_empty((batch, heads, tokens, dim))
    value = torch.empty_like(key)
    try:
        launch(
            index,
            library_for(index).sah_block_cache_read,
            "sah_block_cache_read",
            *cache._pointers(),
            firsts.data_ptr(),
            lengths.data_ptr(),
            key.data_ptr(),
            value.data_ptr(),
            batch,
            heads,
            tokens,
            dim,
            cache.key_codes.shape[0],
            cache.block_table.shape[1],
            dtype_code(tail.dtype),
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP block cache read execution failed") from exc
    return key, value, HIP_BLOCK_CACHE_READ_BACKEND


def _attention_request(
    query: torch.Tensor,
    cache: BlockCache,
    starts: torch.Tensor,
    counts: torch.Tensor | None,
    scale: float | None,
    max_length: int | None,
) -> tuple | None:
    """The library, the device and the query's strides where the attention kernel takes
    the request, else None."""

    tail, size = cache.key_tail, query.shape
    index = tail.get_device()
    if query.dtype is not tail.dtype or len(size) != 4 or query.get_device() != index:
        return None
    batch, kv_heads, _, dim = tail.shape
    if size[0] != batch or size[3] != dim or size[1] < 1 or size[1] % kv_heads:
        return None
    if scale is not None and not abs(scale) <= _MAX_SCALE:
        return None
    if max_length is not None and not (isinstance(max_length, int) and 0 <= max_length <= _MAX_LENGTH):
        return None
    if starts is None or not (_lengths_ok(starts, batch, index) and _lengths_ok(counts, batch, index)):
        return None
    strides, library = _strides(query, size), library_for(index)
    return None if strides is None or library is None else (library, index, strides)


def can_use_hip_block_cache_attention(
    query: torch.Tensor,
    cache: BlockCache,
    starts: torch.Tensor,
    counts: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    max_length: int | None = None,
) -> bool:
    """Whether the attention kernel takes these tensors."""

    return _attention_request(query, cache, starts, counts, scale, max_length) is not None


def hip_block_cache_attention(
    query: torch.Tensor,
    cache: BlockCache,
    starts: torch.Tensor,
    counts: torch.Tensor | None = None,
    *,
    scale: float | None = None,
    max_length: int | None = None,
) -> tuple[torch.Tensor, str]:
    """Causal attention of the new tokens over the cache that holds them already.

    ``query`` is [batch, heads, seq_len, head_dim] (any strides, head_dim
    contiguous), heads a multiple of the cache's: row i of sequence b stands at
    position ``starts[b] + i`` and attends to all positions up to its own, with
    ``starts`` and ``counts`` those of the append.  Returns [batch, seq_len, heads *
    head_dim]; rows from ``counts[b]`` on are zeros.  ``scale`` defaults to
    head_dim ** -0.5 (2 ** 127 is the largest).  ``max_length``, where the program
    knows one, bounds the sequences' lengths below what the table has room for: it
    spares launching the parts of histories that no sequence has.  Longer ones are
    still computed whole.
    """

    request = _attention_request(query, cache, starts, counts, scale, max_length)
    if request is None:
        raise RuntimeError("HIP block cache attention is ineligible for the requested inputs")
    library, index, strides = request
    batch, heads, seq_len, dim = query.shape
    kv_heads, max_blocks = cache.key_tail.shape[1], cache.block_table.shape[1]
    most = min(max_blocks * BLOCK_TOKENS + BLOCK_TOKENS - 1, _MAX_LENGTH if max_length is None else max_length)
    output = query.new_empty((batch, seq_len, heads * dim))
    try:
        size = library.sah_block_cache_attention_workspace_bytes(batch, seq_len, heads, kv_heads, dim, most)
        workspace = torch.empty(size, dtype=torch.uint8, device=query.device) if size else None
        launch(
            index,
            library.sah_block_cache_attention,
            "sah_block_cache_attention",
            query.data_ptr(),
            *cache._pointers(),
            starts.data_ptr(),
            None if counts is None else counts.data_ptr(),
            output.data_ptr(),
            batch,
            heads,
            kv_heads,
            seq_len,
            dim,
            *strides,
            seq_len * heads * dim,
            heads * dim,
            cache.key_codes.shape[0],
            max_blocks,
            most,
            dim**-0.5 if scale is None else float(scale),
            dtype_code(query.dtype),
            None if workspace is None else workspace.data_ptr(),
            size,
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP block cache attention execution failed") from exc
    return output, HIP_BLOCK_CACHE_ATTENTION_BACKEND


__all__ = [
    "BLOCK_TOKENS",
    "BlockCache",
    "HIP_BLOCK_CACHE_APPEND_BACKEND",
    "HIP_BLOCK_CACHE_ATTENTION_BACKEND",
    "HIP_BLOCK_CACHE_READ_BACKEND",
    "SUPPORTED_DTYPES",
    "SUPPORTED_HEAD_DIMS",
    "can_use_hip_block_cache_append",
    "can_use_hip_block_cache_attention",
    "can_use_hip_block_cache_read",
    "hip_block_cache_append",
    "hip_block_cache_attention",
    "hip_block_cache_available",
    "hip_block_cache_read",
]

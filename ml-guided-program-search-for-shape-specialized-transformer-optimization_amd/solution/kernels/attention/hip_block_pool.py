"""Book-keeping of the block cache's places on gfx950: reserving, freeing, forking,
compacting, and the data that moves with it.

No counterpart in the reference.  :class:`BlockPool` holds what the layers of a model share,
the table of the sequences' blocks and a count of each place's holders, on the device:
nothing here waits for the host, so a captured step may hold any of it.  Sequences that
go on from the same tokens share the places of their complete blocks, which are never
written again.

A step with drafts, of ``wanted`` [batch] new tokens (int32, at most ``drafts + 1``), for
every layer::

    missing, _ = hip_block_pool_reserve(pool, starts, drafts + 1, wanted)
    counts = torch.minimum(wanted, 64 * ((starts + wanted) // 64 + 1 - missing) - 1 - starts)
    ...                                            # append, attention, the model's logits
    answer, accepted, _ = hip_verify_draft(logits, tokens, uniforms, draft_logits, counts=counts - 1)
    lengths, ends = starts + counts, starts + 1 + accepted
    for cache in caches:
        hip_block_cache_take_back(cache, lengths, ends)
    hip_block_pool_release(pool, ends)
    starts = ends

``counts`` are the tokens up to the first block that found no place: appended beyond them,
a block is dropped, and with it what the tail held before.  The append and the attention
get them too.  A sequence that can take none (``counts`` 0) takes no part in the
verification (``accepted`` -1), stays where it was and has the same tokens to append in a
later step.

Beams and parallel samples go on from ``sources`` [batch] (int32; a sequence whose source is
outside [0, batch) stays as it is)::

    hip_block_pool_fork(pool, sources, starts)
    for cache in caches:
        hip_block_cache_fork(cache, sources)
    itself = torch.arange(len(sources), device=sources.device)
    starts = starts[torch.where((sources >= 0) & (sources < len(sources)), sources, itself)]

and a pool is compacted, for a smaller one or a copy elsewhere, by::

    origins, used, _ = hip_block_pool_compact(pool)
    for cache in caches:
        hip_block_cache_copy(cache, origins)

csrc/block_pool.hip holds the kernels, include/shape_aware_hip.h the definitions.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from ..hip._library import (
    HipLibraryError,
    dtype_code,
    launch,
    library_available,
    library_for,
)
from .hip_block_cache import BLOCK_TOKENS, BlockCache

HIP_BLOCK_POOL_RESERVE_BACKEND = "hip_block_pool_reserve"
HIP_BLOCK_POOL_RELEASE_BACKEND = "hip_block_pool_release"
HIP_BLOCK_POOL_FORK_BACKEND = "hip_block_pool_fork"
HIP_BLOCK_POOL_COMPACT_BACKEND = "hip_block_pool_compact"
HIP_BLOCK_CACHE_COPY_BACKEND = "hip_block_cache_copy"
HIP_BLOCK_CACHE_FORK_BACKEND = "hip_block_cache_fork"
HIP_BLOCK_CACHE_TAKE_BACK_BACKEND = "hip_block_cache_take_back"

MAX_FORKED_SEQUENCES = 1024
_MAX_TOKENS = 2**31 - 1
_MAX_ENTRIES = 2**31 - 1
_MAX_SEQUENCES = (2**31 - 1) // 1024
_MAX_BLOCKS = (2**31 - 1) // BLOCK_TOKENS  # of a sequence
_MAX_PLACES = 2**31 - 1 - 16384


@dataclass(frozen=True, eq=False)
class BlockPool:
    """Which place holds each block of each sequence, and how many entries name a place.

    ``block_table`` [batch, max_blocks] (int32) is the table of the layers'
    :class:`BlockCache` (-1: no place), ``holders`` [num_blocks] (int32) the number of its
    entries that name a place.  A place without holders is free.
    """

    block_table: torch.Tensor
    holders: torch.Tensor

    def __post_init__(self) -> None:
        table, holders = self.block_table, self.holders
        if table.ndim != 2 or holders.ndim != 1 or table.dtype != torch.int32 or holders.dtype != torch.int32:
            raise ValueError("a pool is block_table [batch, max_blocks] and holders [num_blocks], both int32")
        if not table.is_contiguous() or not holders.is_contiguous() or holders.device != table.device:
            raise ValueError("the pool's tensors must be contiguous and on one device")
        batch, max_blocks = table.shape
        fits = batch <= _MAX_SEQUENCES and max_blocks <= _MAX_BLOCKS and batch * max_blocks <= _MAX_ENTRIES
        # whether the kernels take its sizes (looked at on every call)
        object.__setattr__(self, "_fits", fits and holders.shape[0] <= _MAX_PLACES)

    @classmethod
    def allocate(
        cls, batch: int, *, max_tokens: int, num_blocks: int, device: torch.device | str = "cuda"
    ) -> "BlockPool":
        """A pool of free places, for sequences of up to ``max_tokens``."""

        return cls(
            torch.full((batch, max_tokens // BLOCK_TOKENS), -1, dtype=torch.int32, device=device),
            torch.zeros((num_blocks,), dtype=torch.int32, device=device),
        )

    @classmethod
    def from_table(cls, block_table: torch.Tensor, num_blocks: int) -> "BlockPool":
        """The pool of a table that names places already."""

        places = block_table[(block_table >= 0) & (block_table < num_blocks)].long()
        return cls(block_table, torch.bincount(places, minlength=num_blocks).to(torch.int32))

    @property
    def batch(self) -> int:
        return self.block_table.shape[0]

    @property
    def max_blocks(self) -> int:
        return self.block_table.shape[1]

    @property
    def num_blocks(self) -> int:
        return self.holders.shape[0]


def hip_block_pool_available() -> bool:
    """Whether the gfx950 library loads in this process."""

    return library_available()


def _words_ok(words: torch.Tensor | None, size: int, index: int) -> bool:
    return (
        words is not None
        and words.dtype is torch.int32
        and words.shape == (size,)
        and words.is_contiguous()
        and words.get_device() == index
    )


def _pool_request(pool: BlockPool, words: torch.Tensor | None = None, more: torch.Tensor | None = None) -> tuple | None:
    """The library, the device, batch, max_blocks and num_blocks where the kernels take a
    pool and whole numbers [batch], else None."""

    table = pool.block_table
    index, (batch, max_blocks) = table.get_device(), table.shape
    if not pool._fits:
        return None
    if words is not None and not _words_ok(words, batch, index):
        return None
    if more is not None and not _words_ok(more, batch, index):
        return None
    library = library_for(index)
    return None if library is None else (library, index, batch, max_blocks, pool.holders.shape[0])


def _reserve_request(pool: BlockPool, starts: torch.Tensor, tokens: int, counts: torch.Tensor | None):
    if not isinstance(tokens, int) or isinstance(tokens, bool) or not 0 <= tokens <= _MAX_TOKENS:
        return None
    return None if starts is None else _pool_request(pool, starts, counts)


def can_use_hip_block_pool_reserve(
    pool: BlockPool, starts: torch.Tensor, tokens: int, counts: torch.Tensor | None = None
) -> bool:
    """Whether the reserve kernel takes these tensors."""

    return _reserve_request(pool, starts, tokens, counts) is not None


def hip_block_pool_reserve(
    pool: BlockPool, starts: torch.Tensor, tokens: int, counts: torch.Tensor | None = None
) -> tuple[torch.Tensor, str]:
    """Name a place for every block that appending ``tokens`` rows (``counts[b]`` of them)
    behind ``starts`` completes: the lowest free ones, sequence by sequence.

    Before the append.  Returns ``missing`` [batch] (int32), the blocks that found no free
    place or lie behind the table.  The append drops those with all that they held; of ``n``
    tokens, ``min(n, 64 * ((starts + n) // 64 + 1 - missing) - 1 - starts)`` stay before
    the first of them (where a sequence's entries are named from the front, as these
    calls do).
    """

    request = _reserve_request(pool, starts, tokens, counts)
    if request is None:
        raise RuntimeError("HIP block pool reserve is ineligible for the requested inputs")
    library, index, *sizes = request
    missing = torch.empty_like(starts)
    try:
        size = library.sah_block_pool_reserve_workspace_bytes(*sizes, tokens)
        workspace = starts.new_empty(size // 4)  # 0 bytes without sequences
        launch(
            index,
            library.sah_block_pool_reserve,
            "sah_block_pool_reserve",
            pool.block_table.data_ptr(),
            pool.holders.data_ptr(),
            starts.data_ptr(),
            None if counts is None else counts.data_ptr(),
            missing.data_ptr(),
            *sizes,
            tokens,
            workspace.data_ptr(),
            size,
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP block pool reserve execution failed") from exc
    return missing, HIP_BLOCK_POOL_RESERVE_BACKEND


def can_use_hip_block_pool_release(pool: BlockPool, lengths: torch.Tensor) -> bool:
    """Whether the release kernel takes these tensors."""

    return lengths is not None and _pool_request(pool, lengths) is not None


def hip_block_pool_release(pool: BlockPool, lengths: torch.Tensor) -> str:
    """Give up every block of a sequence but its first ``lengths[b] // 64`` (0 frees a
    sequence that has ended, a negative length leaves it)."""

    request = None if lengths is None else _pool_request(pool, lengths)
    if request is None:
        raise RuntimeError("HIP block pool release is ineligible for the requested inputs")
    library, index, *sizes = request
    try:
        launch(
            index,
            library.sah_block_pool_release,
            "sah_block_pool_release",
            pool.block_table.data_ptr(),
            pool.holders.data_ptr(),
            lengths.data_ptr(),
            *sizes,
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP block pool release execution failed") from exc
    return HIP_BLOCK_POOL_RELEASE_BACKEND


def _fork_request(pool: BlockPool, sources: torch.Tensor, lengths: torch.Tensor) -> tuple | None:
    if sources is None or lengths is None or pool.block_table.shape[0] > MAX_FORKED_SEQUENCES:
        return None
    return _pool_request(pool, sources, lengths)


def can_use_hip_block_pool_fork(pool: BlockPool, sources: torch.Tensor, lengths: torch.Tensor) -> bool:
    """Whether the fork kernel takes these tensors."""

    return _fork_request(pool, sources, lengths) is not None


def hip_block_pool_fork(pool: BlockPool, sources: torch.Tensor, lengths: torch.Tensor) -> str:
    """Let sequence b go on as a copy of sequence ``sources[b]`` of ``lengths[sources[b]]``
    tokens: it gives up its own blocks and shares the source's complete ones.

    All sources are as they were before the call, so sequences may change places; a
    source outside [0, batch), or b itself, leaves b as it is.  Each layer's
    tails follow with :func:`hip_block_cache_fork`.  Up to 1024 sequences.
    """

    request = _fork_request(pool, sources, lengths)
    if request is None:
        raise RuntimeError("HIP block pool fork is ineligible for the requested inputs")
    library, index, *sizes = request
    try:
        launch(
            index,
            library.sah_block_pool_fork,
            "sah_block_pool_fork",
            pool.block_table.data_ptr(),
            pool.holders.data_ptr(),
            sources.data_ptr(),
            lengths.data_ptr(),
            *sizes,
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP block pool fork execution failed") from exc
    return HIP_BLOCK_POOL_FORK_BACKEND


def can_use_hip_block_pool_compact(pool: BlockPool) -> bool:
    """Whether the compaction kernels take this pool."""

    return _pool_request(pool) is not None


def hip_block_pool_compact(pool: BlockPool) -> tuple[torch.Tensor, torch.Tensor, str]:
    """Rename the places in use to the pool's lowest ones: ``(origins, used, marker)``.

    ``origins`` [num_blocks] (int32) names the place whose contents each renamed place
    takes (-1: keeps its own), for :func:`hip_block_cache_copy` of every layer before the
    cache is read or appended to; ``used`` [1] (int32) counts the places in use.
    """

    request = _pool_request(pool)
    if request is None:
        raise RuntimeError("HIP block pool compact is ineligible for the requested inputs")
    library, index, *sizes = request
    origins = torch.empty_like(pool.holders)
    used = pool.holders.new_empty((1,))
    try:
        size = library.sah_block_pool_compact_workspace_bytes(sizes[2])
        workspace = origins.new_empty(size // 4)
        launch(
            index,
            library.sah_block_pool_compact,
            "sah_block_pool_compact",
            pool.block_table.data_ptr(),
            pool.holders.data_ptr(),
            origins.data_ptr(),
            used.data_ptr(),
            *sizes,
            workspace.data_ptr(),
            size,
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP block pool compact execution failed") from exc
    return origins, used, HIP_BLOCK_POOL_COMPACT_BACKEND


def _cache_request(cache: BlockCache, size: int, words: torch.Tensor, more: torch.Tensor | None = None) -> tuple | None:
    """The library and the device where the kernels take a cache and whole numbers
    [size], else None."""

    index = cache.key_tail.get_device()
    if not _words_ok(words, size, index) or (more is not None and not _words_ok(more, size, index)):
        return None
    if not cache._moves:
        return None
    library = library_for(index)
    return None if library is None else (library, index)


def can_use_hip_block_cache_copy(cache: BlockCache, origins: torch.Tensor) -> bool:
    """Whether the copy kernel takes these tensors."""

    return _cache_request(cache, cache.key_codes.shape[0], origins) is not None


def hip_block_cache_copy(cache: BlockCache, origins: torch.Tensor) -> str:
    """Copy complete blocks within the cache: place t takes what place ``origins[t]``
    holds, where that is another place (``origins`` [num_blocks], int32).

    Several places may have one origin.  A place whose origin is itself to be written by
    the call keeps what it holds.
    """

    request = _cache_request(cache, cache.key_codes.shape[0], origins)
    if request is None:
        raise RuntimeError("HIP block cache copy is ineligible for the requested inputs")
    library, index = request
    blocks, heads, _, dim = cache.key_codes.shape
    try:
        launch(
            index,
            library.sah_block_cache_copy,
            "sah_block_cache_copy",
            *cache._pointers()[:4],
            origins.data_ptr(),
            heads,
            dim,
            blocks,
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP block cache copy execution failed") from exc
    return HIP_BLOCK_CACHE_COPY_BACKEND


def _cache_fork_request(cache: BlockCache, sources: torch.Tensor) -> tuple | None:
    batch = cache.key_tail.shape[0]
    return _cache_request(cache, batch, sources) if batch <= MAX_FORKED_SEQUENCES else None


def can_use_hip_block_cache_fork(cache: BlockCache, sources: torch.Tensor) -> bool:
    """Whether the fork kernel takes these tensors."""

    return _cache_fork_request(cache, sources) is not None


def hip_block_cache_fork(cache: BlockCache, sources: torch.Tensor) -> str:
    """Copy the incomplete block of sequence ``sources[b]``, as it was before the call, to
    sequence b, with the sources of :func:`hip_block_pool_fork`."""

    request = _cache_fork_request(cache, sources)
    if request is None:
        raise RuntimeError("HIP block cache fork is ineligible for the requested inputs")
    library, index = request
    batch, heads, _, dim = cache.key_tail.shape
    try:
        launch(
            index,
            library.sah_block_cache_fork,
            "sah_block_cache_fork",
            cache.key_tail.data_ptr(),
            cache.value_tail.data_ptr(),
            sources.data_ptr(),
            batch,
            heads,
            dim,
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP block cache fork execution failed") from exc
    return HIP_BLOCK_CACHE_FORK_BACKEND


def _take_back_request(cache: BlockCache, lengths: torch.Tensor, ends: torch.Tensor) -> tuple | None:
    if ends is None or not cache._goes_back:
        return None
    return _cache_request(cache, cache.key_tail.shape[0], lengths, ends)


def can_use_hip_block_cache_take_back(cache: BlockCache, lengths: torch.Tensor, ends: torch.Tensor) -> bool:
    """Whether the take-back kernel takes these tensors."""

    return _take_back_request(cache, lengths, ends) is not None


def hip_block_cache_take_back(cache: BlockCache, lengths: torch.Tensor, ends: torch.Tensor) -> str:
    """Make sequences of ``lengths[b]`` tokens ready to go on from ``ends[b]``, anywhere
    up to that.

    Where ``ends[b]`` falls into a complete block, the tail takes that block's values
    back: its codes times their scale, so these tokens are coded a second time once
    their block is complete again.  Call it before the block's place is released or
    written; ``starts = ends`` from then on.
    """

    tail = cache.key_tail
    batch, heads, _, dim = tail.shape
    request = _take_back_request(cache, lengths, ends)
    if request is None:
        raise RuntimeError("HIP block cache take back is ineligible for the requested inputs")
    library, index = request
    try:
        launch(
            index,
            library.sah_block_cache_take_back,
            "sah_block_cache_take_back",
            *cache._pointers(),
            lengths.data_ptr(),
            ends.data_ptr(),
            batch,
            heads,
            dim,
            cache.key_codes.shape[0],
            cache.block_table.shape[1],
            dtype_code(tail.dtype),
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP block cache take back execution failed") from exc
    return HIP_BLOCK_CACHE_TAKE_BACK_BACKEND


__all__ = [
    "BlockPool",
    "HIP_BLOCK_CACHE_COPY_BACKEND",
    "HIP_BLOCK_CACHE_FORK_BACKEND",
    "HIP_BLOCK_CACHE_TAKE_BACK_BACKEND",
    "HIP_BLOCK_POOL_COMPACT_BACKEND",
    "HIP_BLOCK_POOL_FORK_BACKEND",
    "HIP_BLOCK_POOL_RELEASE_BACKEND",
    "HIP_BLOCK_POOL_RESERVE_BACKEND",
    "MAX_FORKED_SEQUENCES",
    "can_use_hip_block_cache_copy",
    "can_use_hip_block_cache_fork",
    "can_use_hip_block_cache_take_back",
    "can_use_hip_block_pool_compact",
    "can_use_hip_block_pool_fork",
    "can_use_hip_block_pool_release",
    "can_use_hip_block_pool_reserve",
    "hip_block_cache_copy",
    "hip_block_cache_fork",
    "hip_block_cache_take_back",
    "hip_block_pool_available",
    "hip_block_pool_compact",
    "hip_block_pool_fork",
    "hip_block_pool_release",
    "hip_block_pool_reserve",
]

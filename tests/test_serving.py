"""The operators around a decoding step with drafts, without a GPU: refusals of the C
entries before any launch, workspace sizes, eligibility in Python and the checks of the
pool's and the adapters' own tensors."""

from __future__ import annotations

import re
import sys
import textwrap
from pathlib import Path

import pytest
import torch

from serving_reference import Book, TokenCache
from solution.kernels.attention import hip_block_pool as pool_module
from solution.kernels.attention import (
    BlockCache,
    BlockPool,
    can_use_hip_block_cache_copy,
    can_use_hip_block_pool_reserve,
    hip_block_cache_copy,
    hip_block_cache_fork,
    hip_block_cache_take_back,
    hip_block_pool_compact,
    hip_block_pool_fork,
    hip_block_pool_release,
    hip_block_pool_reserve,
)
from solution.kernels.hip import _library
from solution.kernels.projection import LowRankAdapters, can_use_hip_low_rank_adapters, hip_low_rank_adapters
from solution.kernels.projection import hip_low_rank as low_rank_module
from solution.kernels.sampling import can_use_hip_verify_draft, hip_verify_draft

# An address that the host checks may look at and no kernel reads: every call below is
# refused, or has nothing to do, before a launch.
P = 0x10000
BF16, F16, F32 = 2, 1, 0
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 4


def _call(name, defaults, **changes):
    unknown = set(changes) - set(defaults)
    assert not unknown, unknown
    return getattr(_library.load_library(), name)(*{**defaults, **changes}.values())


VERIFY = dict(
    target=P, draft=P, tokens=P, uniforms=P, counts=None, temperatures=None, answer=P, accepted=P, batch=2, drafts=3,
    vocab=1000, t_sb=4000, t_ss=1000, d_sb=3000, d_ss=1000, dtype=BF16, workspace=P, workspace_bytes=0, stream=None,
)


@pytest.mark.parametrize(
    "changes,status",
    [
        ({"batch": 0}, OK),
        ({}, WORKSPACE),
        ({"workspace": None, "workspace_bytes": 1 << 20}, WORKSPACE),
        ({"workspace": P + 8, "workspace_bytes": 1 << 20}, INVALID),
        ({"dtype": 7}, INVALID),
        ({"batch": -1}, INVALID),
        ({"drafts": -1}, INVALID),
        ({"vocab": 0}, INVALID),
        ({"drafts": 1025}, UNSUPPORTED),
        ({"vocab": 2**31 - 1}, UNSUPPORTED),
        ({"batch": 1 << 20, "vocab": 1 << 20}, UNSUPPORTED),
        ({"target": None}, INVALID),
        ({"tokens": None}, INVALID),
        ({"uniforms": None}, INVALID),
        ({"answer": None}, INVALID),
        ({"accepted": None}, INVALID),
        ({"target": P + 1}, INVALID),
        ({"dtype": F32, "draft": P + 2}, INVALID),
        ({"tokens": P + 4}, INVALID),
        ({"counts": P + 2}, INVALID),
        ({"temperatures": P + 1}, INVALID),
        ({"drafts": 0, "tokens": None}, WORKSPACE),
    ],
)
def test_verify_entry_refuses_before_launch(changes, status):
    assert _call("sah_verify_draft", VERIFY, **changes) == status


def test_verify_workspace_sizes():
    size = _library.load_library().sah_verify_draft_workspace_bytes
    assert size(0, 3, 1000, 1) == size(2, 1025, 1000, 1) == size(2, 3, 0, 1) == size(-1, 3, 1000, 1) == 0
    # 16 bytes a row and 8192 logits of it, 40 bytes a request and 2048 logits, 40 a request
    assert size(2, 3, 1000, 1) == 2 * (7 * 16 + 40 + 40)
    assert size(2, 3, 8193, 0) == 2 * (4 * 2 * 16 + 5 * 40 + 40)


ADAPTERS = dict(
    x=P, base=P, down=P, up=P, scales=None, ranks=None, indices=P, counts=None, y=P, batch=2, seq_len=3, in_features=4096,
    out_features=32, adapters=4, rank=16, x_sb=12288, x_ss=4096, p_sb=96, p_ss=32, y_sb=96, y_ss=32, dtype=BF16,
    workspace=P, workspace_bytes=0, stream=None,
)


@pytest.mark.parametrize(
    "changes,status",
    [
        ({"batch": 0}, OK),
        ({"seq_len": 0}, OK),
        ({}, WORKSPACE),
        ({"workspace": P + 4, "workspace_bytes": 1 << 20}, INVALID),
        ({"dtype": F32}, UNSUPPORTED),
        ({"batch": -1}, INVALID),
        ({"rank": 0}, INVALID),
        ({"rank": 12}, UNSUPPORTED),
        ({"rank": 136}, UNSUPPORTED),
        ({"in_features": 60}, UNSUPPORTED),
        ({"out_features": 36}, UNSUPPORTED),
        ({"in_features": 0}, INVALID),
        ({"adapters": -1}, INVALID),
        ({"x": None}, INVALID),
        ({"down": None}, INVALID),
        ({"indices": None}, INVALID),
        ({"up": P + 8}, INVALID),
        ({"base": P + 2}, INVALID),
        ({"scales": P + 2}, INVALID),
        ({"indices": P + 1}, INVALID),
        ({"x_ss": 68}, INVALID),
        ({"p_sb": 100}, INVALID),
        # rows of y that overlap
        ({"y_ss": 0}, INVALID),
        ({"y_ss": 24}, INVALID),
        ({"y_sb": 88}, INVALID),
        ({"y_sb": 0, "y_ss": 64}, INVALID),
        ({"y_sb": -96}, INVALID),
        # tokens outermost is a layout
        ({"y_sb": 32, "y_ss": 64}, WORKSPACE),
        ({"y_sb": 32, "y_ss": 56}, INVALID),
        ({"batch": 1 << 20, "seq_len": 1 << 20}, INVALID),
        ({"batch": 1 << 20, "seq_len": 1 << 20, "y_sb": 1 << 25}, UNSUPPORTED),
    ],
)
def test_adapters_entry_refuses_before_launch(changes, status):
    assert _call("sah_low_rank_adapters", ADAPTERS, **changes) == status


def test_adapters_workspace_sizes():
    size = _library.load_library().sah_low_rank_adapters_workspace_bytes
    assert size(0, 1, 64, 64, 16) == size(1, 0, 64, 64, 16) == size(1, 1, 64, 64, 12) == size(1, 1, 60, 64, 16) == 0
    few = size(1, 1, 4096, 4096, 64)
    assert few > 0 and few % (64 * 16 * 4) == 0
    assert size(64, 20000, 4096, 4096, 64) == size(1, 1, 1024, 1024, 16) == 0
    assert size(64, 1, 1024, 4096, 16) > 0


POOL = dict(table=P, holders=P)
SIZES = dict(batch=2, max_blocks=4, num_blocks=10)
RESERVE = dict(**POOL, starts=P, counts=None, missing=P, **SIZES, tokens=5, workspace=P, workspace_bytes=0, stream=None)
RELEASE = dict(**POOL, lengths=P, **SIZES, stream=None)
FORK = dict(**POOL, sources=P, lengths=P, **SIZES, stream=None)
COMPACT = dict(**POOL, origins=P, used=P, **SIZES, workspace=P, workspace_bytes=0, stream=None)
OF_POOL = [
    ({"batch": -1}, INVALID),
    ({"batch": 1 << 22}, INVALID),
    ({"max_blocks": -1}, INVALID),
    ({"max_blocks": 1 << 26}, INVALID),
    ({"num_blocks": -1}, INVALID),
    ({"num_blocks": 2**31 - 1}, INVALID),
    ({"batch": 1 << 16, "max_blocks": 1 << 15}, UNSUPPORTED),
    ({"table": None}, INVALID),
    ({"holders": None}, INVALID),
    ({"table": P + 2}, INVALID),
    ({"holders": P + 1}, INVALID),
]


@pytest.mark.parametrize(
    "changes,status",
    OF_POOL
    + [
        ({"batch": 0}, OK),
        ({}, WORKSPACE),
        ({"workspace": P + 2, "workspace_bytes": 1 << 20}, INVALID),
        ({"tokens": -1}, INVALID),
        ({"tokens": 1 << 31}, INVALID),
        ({"starts": None}, INVALID),
        ({"missing": None}, INVALID),
        ({"counts": P + 2}, INVALID),
    ],
)
def test_reserve_entry_refuses_before_launch(changes, status):
    assert _call("sah_block_pool_reserve", RESERVE, **changes) == status


@pytest.mark.parametrize(
    "changes,status",
    OF_POOL
    + [
        ({"batch": 0}, OK),
        ({"max_blocks": 0}, OK),
        ({"lengths": None}, INVALID),
        ({"lengths": P + 2}, INVALID),
    ],
)
def test_release_entry_refuses_before_launch(changes, status):
    assert _call("sah_block_pool_release", RELEASE, **changes) == status


@pytest.mark.parametrize(
    "changes,status",
    OF_POOL
    + [
        ({"batch": 0}, OK),
        ({"max_blocks": 0}, OK),
        ({"batch": 1025}, UNSUPPORTED),
        ({"sources": None}, INVALID),
        ({"lengths": P + 2}, INVALID),
    ],
)
def test_fork_entry_refuses_before_launch(changes, status):
    assert _call("sah_block_pool_fork", FORK, **changes) == status


@pytest.mark.parametrize(
    "changes,status",
    OF_POOL
    + [
        ({}, WORKSPACE),
        ({"workspace": None, "workspace_bytes": 1 << 20}, WORKSPACE),
        ({"workspace": P + 2, "workspace_bytes": 1 << 20}, INVALID),
        ({"num_blocks": 0, "origins": None}, WORKSPACE),
        ({"origins": None}, INVALID),
        ({"used": None}, INVALID),
    ],
)
def test_compact_entry_refuses_before_launch(changes, status):
    assert _call("sah_block_pool_compact", COMPACT, **changes) == status


def test_pool_workspace_sizes():
    library = _library.load_library()
    size = library.sah_block_pool_reserve_workspace_bytes
    assert size(0, 4, 10, 5) == size(2, 4, 10, -1) == 0
    assert size(2, 4, 10, 5) == (2 + 2) * 4  # a block each
    assert size(2, 4, 10, 1000) == (2 + 8) * 4  # no more than the table's
    assert size(5, 4, 10, 1000) == (5 + 10) * 4  # no more than there are
    assert size(5, 0, 10, 1000) == 5 * 4
    assert library.sah_block_pool_compact_workspace_bytes(10) == (6 + 6 + 10 + 1) * 4
    assert library.sah_block_pool_compact_workspace_bytes(0) > 0
    assert library.sah_block_pool_compact_workspace_bytes(-1) == 0


CODES = dict(key_codes=P, value_codes=P, key_scales=P, value_scales=P)
COPY = dict(**CODES, origins=P, kv_heads=2, head_dim=64, num_blocks=4, stream=None)
TAILS = dict(key_tail=P, value_tail=P, sources=P, batch=2, kv_heads=2, head_dim=64, stream=None)
TAKE = dict(
    **CODES, key_tail=P, value_tail=P, table=P, lengths=P, ends=P, batch=2, kv_heads=2, head_dim=64, num_blocks=4,
    max_blocks=2, dtype=BF16, stream=None,
)


@pytest.mark.parametrize(
    "changes,status",
    [
        ({"num_blocks": 0}, OK),
        ({"num_blocks": -1}, INVALID),
        ({"head_dim": 96}, UNSUPPORTED),
        ({"kv_heads": 0}, INVALID),
        ({"key_codes": None}, INVALID),
        ({"value_scales": None}, INVALID),
        ({"origins": None}, INVALID),
        ({"value_codes": P + 8}, INVALID),
        ({"origins": P + 2}, INVALID),
    ],
)
def test_copy_entry_refuses_before_launch(changes, status):
    assert _call("sah_block_cache_copy", COPY, **changes) == status


@pytest.mark.parametrize(
    "changes,status",
    [
        ({"batch": 0}, OK),
        ({"batch": -1}, INVALID),
        ({"batch": 1025}, UNSUPPORTED),
        ({"head_dim": 32}, UNSUPPORTED),
        ({"kv_heads": 65537}, INVALID),
        ({"key_tail": None}, INVALID),
        ({"value_tail": P + 8}, INVALID),
        ({"sources": None}, INVALID),
        ({"sources": P + 1}, INVALID),
    ],
)
def test_tail_fork_entry_refuses_before_launch(changes, status):
    assert _call("sah_block_cache_fork", TAILS, **changes) == status


@pytest.mark.parametrize(
    "changes,status",
    [
        ({"batch": 0}, OK),
        ({"batch": -1}, INVALID),
        ({"dtype": F32}, UNSUPPORTED),
        ({"head_dim": 96}, UNSUPPORTED),
        ({"kv_heads": 0}, INVALID),
        ({"num_blocks": -1}, INVALID),
        ({"max_blocks": -1}, INVALID),
        ({"lengths": None}, INVALID),
        ({"ends": P + 2}, INVALID),
        ({"key_tail": None}, INVALID),
        ({"table": None}, INVALID),
        ({"key_scales": None}, INVALID),
        ({"value_tail": P + 4}, INVALID),
        ({"value_scales": P + 2}, INVALID),
        ({"batch": 1 << 30}, UNSUPPORTED),
    ],
)
def test_take_back_entry_refuses_before_launch(changes, status):
    assert _call("sah_block_cache_take_back", TAKE, **changes) == status


def test_pool_allocation():
    pool = BlockPool.allocate(3, max_tokens=200, num_blocks=7, device="cpu")
    assert (pool.batch, pool.max_blocks, pool.num_blocks) == (3, 3, 7)
    assert pool.block_table.eq(-1).all() and pool.holders.eq(0).all()
    cache = BlockCache.allocate(3, 2, 64, max_tokens=200, num_blocks=7, block_table=pool.block_table, device="cpu")
    assert cache.block_table is pool.block_table
    table = torch.tensor([[0, 3, -1], [0, 5, 9]], dtype=torch.int32)
    assert BlockPool.from_table(table, 6).holders.tolist() == [2, 0, 0, 1, 0, 1]  # 9 is no place of 6


@pytest.mark.parametrize(
    "name,make",
    [
        ("block_table", lambda t: t.long()),
        ("block_table", lambda t: t[0]),
        ("block_table", lambda t: t[:, :2]),
        ("holders", lambda t: t.long()),
        ("holders", lambda t: t[:, None]),
        ("holders", lambda t: t[::2]),
    ],
)
def test_pool_of_tensors_that_do_not_belong_together(name, make):
    pool = BlockPool.allocate(3, max_tokens=200, num_blocks=7, device="cpu")
    parts = {"block_table": pool.block_table, "holders": pool.holders}
    parts[name] = make(parts[name])
    with pytest.raises(ValueError):
        BlockPool(**parts)


def _adapter_parts():
    return {
        "down": torch.zeros(3, 16, 64, dtype=torch.bfloat16),
        "up": torch.zeros(3, 32, 16, dtype=torch.bfloat16),
        "scales": torch.ones(3),
        "ranks": torch.full((3,), 16, dtype=torch.int32),
    }


@pytest.mark.parametrize(
    "name,make",
    [
        ("down", lambda t: t.half()),
        ("down", lambda t: t.float()),
        ("down", lambda t: t[0]),
        ("down", lambda t: t[:2].contiguous()),
        ("down", lambda t: t[..., :60].contiguous()),
        ("down", lambda t: t[:, :, :32]),
        ("up", lambda t: t[:, :, :8].contiguous()),
        ("up", lambda t: t[:, :30].contiguous()),
        ("up", lambda t: t[:, :0].contiguous()),
        ("scales", lambda t: t.double()),
        ("scales", lambda t: t[:2]),
        ("ranks", lambda t: t.long()),
        ("down", lambda t: t.requires_grad_()),
    ],
)
def test_adapters_of_tensors_that_do_not_belong_together(name, make):
    parts = _adapter_parts()
    LowRankAdapters(**parts)
    parts[name] = make(parts[name])
    with pytest.raises(ValueError):
        LowRankAdapters(**parts)


def test_adapters_of_ranks_that_no_kernel_takes():
    for rank in (12, 136):
        with pytest.raises(ValueError):
            LowRankAdapters(torch.zeros(1, rank, 64, dtype=torch.float16), torch.zeros(1, 32, rank, dtype=torch.float16))


def test_packed_adapters():
    generator = torch.Generator().manual_seed(3)
    given = [
        (torch.randn(r, 24, generator=generator).half(), torch.randn(16, r, generator=generator).half(), s)
        for r, s in ((5, 0.5), (12, 2.0), (1, 1.0))
    ]
    packed = LowRankAdapters.pack(given)
    assert (packed.rank, packed.in_features, packed.out_features) == (16, 24, 16)
    assert packed.ranks.tolist() == [5, 12, 1] and packed.scales.tolist() == [0.5, 2.0, 1.0]
    for place, (down, up, _) in enumerate(given):
        r = down.shape[0]
        assert torch.equal(packed.down[place, :r], down) and packed.down[place, r:].eq(0).all()
        assert torch.equal(packed.up[place, :, :r], up) and packed.up[place, :, r:].eq(0).all()
    for bad in (
        [],
        [(given[0][0], given[1][1], 1.0)],
        [given[0], (given[1][0][:, :16], given[1][1], 1.0)],
        [given[0], (given[1][0].bfloat16(), given[1][1], 1.0)],
        [(torch.zeros(129, 24).half(), torch.zeros(16, 129).half(), 1.0)],
    ):
        with pytest.raises(ValueError):
            LowRankAdapters.pack(bad)


@pytest.mark.parametrize(
    "make,want",
    [
        (lambda t: t, (64, 16)),
        (lambda t: t[:, :1], (64, 0)),
        (lambda t: t[:1], (0, 16)),
        (lambda t: t.transpose(0, 1), (16, 64)),
        (lambda t: t[..., 8:], (64, 16)),
        (lambda t: t[..., 4:12], None),  # off the multiples of 16 bytes
        (lambda t: t.transpose(1, 2), None),
        (lambda t: t[:, 0], (64, 0)),
    ],
)
def test_adapter_rows_that_are_read_in_place(make, want):
    assert low_rank_module._strides(make(torch.zeros(3, 4, 16, dtype=torch.bfloat16))) == want


def test_adapter_outputs_apart_from_inputs():
    store = torch.zeros(2, 3, 64, dtype=torch.bfloat16)
    assert low_rank_module._apart(store[0], store[1])
    assert not low_rank_module._apart(store[:, 0], store[:, 1])  # rows of one lie between the other's
    assert not low_rank_module._apart(store, store[1])
    assert low_rank_module._apart(store[:0], store)


@pytest.fixture
def any_device(monkeypatch):
    """The library for tensors without storage, whose sizes alone are looked at: on the
    device "meta", no call beyond the predicates."""

    verify_module = sys.modules[hip_verify_draft.__module__]
    for module in (verify_module, low_rank_module, pool_module):
        monkeypatch.setattr(module, "library_for", lambda index: _library.load_library())


def _meta(*shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize(
    "batch,drafts,vocab,sampled,taken",
    [
        ((2**32 - 1) // 1024, 0, 2, False, True),
        ((2**32 - 1) // 1024 + 1, 0, 2, False, False),
        ((2**32 - 1) // 1024 // 2049, 1024, 100, True, True),
        ((2**32 - 1) // 1024 // 2049 + 1, 1024, 100, True, False),
        (1, 0, 2**31 - 1 - 8192, False, True),
        (1, 0, 2**31 - 8192, False, False),
        (1, 1025, 100, False, False),
        (0, 3, 100, True, True),
    ],
)
def test_verify_predicate_at_the_entry_s_limits(any_device, batch, drafts, vocab, sampled, taken):
    target, draft = (_meta(batch, n, vocab, dtype=torch.bfloat16) for n in (drafts + 1, drafts))
    tokens, uniforms = _meta(batch, drafts, dtype=torch.int64), _meta(batch, drafts + 1, dtype=torch.float32)
    assert can_use_hip_verify_draft(target, tokens, uniforms, draft if sampled else None) == taken
    if not taken:
        sizes = dict(batch=batch, drafts=drafts, vocab=vocab, draft=P if sampled else None)
        assert _call("sah_verify_draft", VERIFY, **sizes, workspace_bytes=1 << 40) == UNSUPPORTED


@pytest.mark.parametrize(
    "batch,seq,k,n,taken",
    [
        (1, 1, 2**24, 8, True),
        (1, 1, 2**24 + 8, 8, False),
        (1, 1, 8, 2**24, True),
        (1, 1, 8, 2**24 + 8, False),
        ((2**32 - 1) // 256, 1, 8, 8, True),
        ((2**32 - 1) // 256 + 1, 1, 8, 8, False),
        (1, 16 * ((2**32 - 1) // 256 // 3), 8, 136, True),
        (1, 16 * ((2**32 - 1) // 256 // 3) + 1, 8, 136, False),
    ],
)
def test_adapters_predicate_at_the_entry_s_limits(any_device, batch, seq, k, n, taken):
    down, up = _meta(1, 8, k, dtype=torch.bfloat16), _meta(1, n, 8, dtype=torch.bfloat16)
    value, projected = _meta(batch, seq, k, dtype=torch.bfloat16), _meta(batch, seq, n, dtype=torch.bfloat16)
    if max(k, n) > 2**24:
        with pytest.raises(ValueError, match="at most"):
            LowRankAdapters(down, up)
    else:
        assert can_use_hip_low_rank_adapters(value, projected, LowRankAdapters(down, up), _meta(batch)) == taken
    if not taken:
        sizes = dict(batch=batch, seq_len=seq, in_features=k, out_features=n, adapters=1, rank=8)
        rows = dict(x_sb=seq * k, x_ss=k, p_sb=seq * n, p_ss=n, y_sb=seq * n, y_ss=n)
        assert _call("sah_low_rank_adapters", ADAPTERS, **sizes, **rows, workspace_bytes=1 << 40) == UNSUPPORTED


@pytest.mark.parametrize(
    "batch,max_blocks,num_blocks,taken",
    [
        (2097151, 1, 5, True),
        (2097152, 1, 5, False),
        (1, 2**25 - 1, 5, True),
        (1, 2**25, 5, False),
        (65536, 32767, 5, True),
        (65536, 32768, 5, False),
        (2, 3, 2**31 - 1 - 16384, True),
        (2, 3, 2**31 - 16384, False),
    ],
)
def test_pool_predicates_at_the_entries_limits(any_device, batch, max_blocks, num_blocks, taken):
    pool, words = BlockPool(_meta(batch, max_blocks), _meta(num_blocks)), _meta(batch)
    assert can_use_hip_block_pool_reserve(pool, words, 3) == taken
    assert pool_module.can_use_hip_block_pool_release(pool, words) == taken
    assert pool_module.can_use_hip_block_pool_compact(pool) == taken
    assert pool_module.can_use_hip_block_pool_fork(pool, words, words) == (taken and batch <= 1024)
    if not taken:
        sizes = dict(batch=batch, max_blocks=max_blocks, num_blocks=num_blocks)
        for name, defaults in (("reserve", RESERVE), ("release", RELEASE), ("fork", FORK), ("compact", COMPACT)):
            more = {"workspace_bytes": 1 << 40} if "workspace" in defaults else {}
            assert _call("sah_block_pool_" + name, defaults, **sizes, **more) in (INVALID, UNSUPPORTED)


@pytest.mark.parametrize(
    "batch,heads,blocks,width,taken",
    [
        (2, 65536, 5, 3, (True, True, True)),
        (2, 65537, 5, 3, (False, False, False)),
        (1025, 2, 5, 3, (True, False, True)),
        ((2**32 - 1) // 256 // 4, 2, 5, 3, (True, False, True)),
        ((2**32 - 1) // 256 // 4 + 1, 2, 5, 3, (True, False, False)),
        (1, 1, 2**31 - 1, 3, (True, True, True)),
        (1, 1, 2**31, 3, (False, False, False)),
        (1, 1, 5, 2**25 - 1, (True, True, True)),
        (1, 1, 5, 2**25, (True, True, False)),
    ],
)
def test_cache_predicates_at_the_entries_limits(any_device, batch, heads, blocks, width, taken):
    """Of the copy, the tails' fork and the take-back."""

    codes, scales = _meta(blocks, heads, 64, 64, dtype=torch.uint8), _meta(blocks, heads, dtype=torch.float32)
    tail = _meta(batch, heads, 64, 64, dtype=torch.bfloat16)
    cache, words = BlockCache(codes, codes, scales, scales, tail, tail, _meta(batch, width)), _meta(batch)
    got = (
        can_use_hip_block_cache_copy(cache, _meta(blocks)),
        pool_module.can_use_hip_block_cache_fork(cache, words),
        pool_module.can_use_hip_block_cache_take_back(cache, words, words),
    )
    assert got == taken
    refused = (INVALID, UNSUPPORTED)
    if not taken[0]:
        assert _call("sah_block_cache_copy", COPY, kv_heads=heads, num_blocks=blocks) in refused
    if not taken[1] and blocks <= 2**31 - 1:
        assert _call("sah_block_cache_fork", TAILS, batch=batch, kv_heads=heads) in refused
    if not taken[2]:
        sizes = dict(batch=batch, kv_heads=heads, num_blocks=blocks, max_blocks=width)
        assert _call("sah_block_cache_take_back", TAKE, **sizes) in refused


def test_operators_refuse_cpu_tensors():
    pool = BlockPool.allocate(2, max_tokens=200, num_blocks=7, device="cpu")
    cache = BlockCache.allocate(2, 2, 64, max_tokens=200, num_blocks=7, block_table=pool.block_table, device="cpu")
    words = torch.zeros(2, dtype=torch.int32)
    origins = torch.full((7,), -1, dtype=torch.int32)
    assert not can_use_hip_block_pool_reserve(pool, words, 3) and not can_use_hip_block_cache_copy(cache, origins)
    adapters = LowRankAdapters(**_adapter_parts())
    value, projected = torch.zeros(2, 1, 64).bfloat16(), torch.zeros(2, 1, 32).bfloat16()
    assert not can_use_hip_low_rank_adapters(value, projected, adapters, words)
    logits, tokens, uniforms = torch.zeros(2, 4, 10), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 4)
    assert not can_use_hip_verify_draft(logits, tokens, uniforms)
    calls = (
        lambda: hip_block_pool_reserve(pool, words, 3),
        lambda: hip_block_pool_release(pool, words),
        lambda: hip_block_pool_fork(pool, words, words),
        lambda: hip_block_pool_compact(pool),
        lambda: hip_block_cache_copy(cache, origins),
        lambda: hip_block_cache_fork(cache, words),
        lambda: hip_block_cache_take_back(cache, words, words),
        lambda: hip_low_rank_adapters(value, projected, adapters, words),
        lambda: hip_verify_draft(logits, tokens, uniforms),
    )
    for call in calls:
        with pytest.raises(RuntimeError, match="ineligible"):
            call()
    assert pool.block_table.eq(-1).all()


# ---------------------------------------------------------------------------
# the documented recipes, run on whole numbers


def _recipes(where):
    """The documented calls for the block pool, as texts: a step's before and after the
    model's own part, and what follows them."""

    if where == "docstring":
        blocks = re.findall(r"::\n\n((?:    .*\n|\n)+)", pool_module.__doc__)
        text = "\n".join(textwrap.dedent(block) for block in blocks)
    else:
        documents = [path.read_text() for path in Path(__file__).resolve().parents[1].glob("*.md")]
        blocks = [block for document in documents for block in re.findall(r"```python\n(.*?)```", document, re.S)]
        (text,) = [block for block in blocks if "hip_block_pool_reserve(pool" in block]
        text = text[re.search(r"^.*hip_block_pool_reserve\(pool", text, re.M).start() :]
    before, rest = text.split("\n...", 1)
    after, others = rest[rest.index("answer, accepted") :].split("starts = ends\n", 1)
    return before, after + "starts = ends\n", others


def _words(values):
    return torch.tensor(values, dtype=torch.int32)


def _stand_ins(book, caches, accepts):
    """The calls that the recipes make, on a book and caches of whole numbers; ``accepts``
    says how many drafts of a request stand at most."""

    def reserve(pool, starts, tokens, counts=None):
        return _words(book.reserve(starts.tolist(), tokens, None if counts is None else counts.tolist())), "marker"

    def verify(logits, tokens, uniforms, draft=None, *, counts=None, temperatures=None):
        count = [tokens.shape[1]] * tokens.shape[0] if counts is None else counts.tolist()
        return tokens, _words([-1 if c < 0 else min(c, a) for c, a in zip(count, accepts)]), "marker"

    def compact(pool):
        origins, used = book.compact()
        return _words(origins), _words([used]), "marker"

    return dict(
        torch=torch, pool=book, caches=caches, logits=None, uniforms=None, draft_logits=None, temperatures=None,
        hip_block_pool_reserve=reserve,
        hip_verify_draft=verify,
        hip_block_cache_take_back=lambda cache, lengths, ends: cache.take_back(lengths.tolist(), ends.tolist()),
        hip_block_pool_release=lambda pool, lengths: book.release(lengths.tolist()),
        hip_block_pool_fork=lambda pool, sources, lengths: book.fork(sources.tolist(), lengths.tolist()),
        hip_block_cache_fork=lambda cache, sources: cache.fork(sources.tolist()),
        hip_block_pool_compact=compact,
        hip_block_cache_copy=lambda cache, origins: cache.copy(origins.tolist()),
    )


@pytest.mark.parametrize("where", ["docstring", "guide"])
@pytest.mark.parametrize("blocks", [0, 1, 2, 3, 5, 30])
def test_documented_step_keeps_its_tokens_where_places_run_out(where, blocks):
    """Steps of sequences that ask for fewer and for more places than there are: whatever
    was kept is held, and a sequence goes on wherever its next token needs no block."""

    before, after, _ = _recipes(where)
    drafts, starts = 7, [60, 57, 63, 0, 126, 10]
    width = 4
    book = Book([[-1] * width for _ in starts], [0] * (blocks + 2))
    cache = TokenCache(book)
    book.table[4][0], book.holders[0] = 0, 1  # one sequence has a block
    book.holders[1] = 1  # and one place is someone else's
    kept = [[1000 * b + i for i in range(n)] for b, n in enumerate(starts)]
    cache.append([0] * len(starts), starts, kept)
    wants = [8, 8, 8, 8, 8, 3]
    accepts = [7, 2, 0, 7, 5, 1]
    names = _stand_ins(book, [cache], accepts) | dict(drafts=drafts, starts=_words(starts))
    for step in range(40):
        names |= dict(wanted=_words(wants), tokens=torch.zeros((len(starts), drafts), dtype=torch.int64))
        now = names["starts"].tolist()
        fresh = [[100_000 * (step + 1) + 1000 * b + i for i in range(drafts + 1)] for b in range(len(starts))]
        exec(before, names)
        counts = names["counts"].tolist() if "counts" in names else [drafts + 1] * len(starts)
        cache.append(now, counts, fresh)
        exec(after, names)
        for b, (start, end) in enumerate(zip(now, names["starts"].tolist())):
            assert start <= end <= start + wants[b]
            if start % 64 < 63:  # its next token fits the tail
                assert end > start or start >= 64 * width + 63
            kept[b] = kept[b] + fresh[b][: end - start]
            assert cache.read(b, end) == kept[b], (step, b)


@pytest.mark.parametrize("where", ["docstring", "guide"])
@pytest.mark.parametrize("sources", [[1, 0, -1, 3, 7, 0], [-1] * 6, [6, 6, 6, 0, 0, 0], [5, 4, 3, 2, 1, 0]])
def test_documented_beams_go_on_where_their_sources_were(where, sources):
    """Behind a step whose drafts stood in part: every sequence holds what its source
    held, as long as that was, and goes on from there; so it does after the compaction."""

    before, after, others = _recipes(where)
    drafts, first = 7, [60, 130, 64, 5, 200, 127]
    batch, width = len(first), 5
    book = Book([[-1] * width for _ in first], [0] * 40)
    cache = TokenCache(book)
    kept = [[1000 * b + i for i in range(n)] for b, n in enumerate(first)]
    names = _stand_ins(book, [cache], [7, 2, 0, 7, 5, 1]) | dict(drafts=drafts)
    book.reserve([0] * batch, max(first), first)
    cache.append([0] * batch, first, kept)
    names |= dict(starts=_words(first), wanted=_words([8] * batch), tokens=torch.zeros((batch, drafts), dtype=torch.int64))
    fresh = [[100_000 + 1000 * b + i for i in range(drafts + 1)] for b in range(batch)]
    exec(before, names)
    cache.append(first, [drafts + 1] * batch, fresh)
    exec(after, names)
    kept = [kept[b] + fresh[b][: n - first[b]] for b, n in enumerate(names["starts"].tolist())]
    names["sources"] = _words(sources)
    names["lengths"] = names["lengths"].clone()
    exec(others, names)
    want = [kept[s if 0 <= s < batch else b] for b, s in enumerate(sources)]
    assert names["starts"].tolist() == [len(tokens) for tokens in want]
    for b, tokens in enumerate(want):
        assert cache.read(b, len(tokens)) == tokens
        # nothing is named behind what is held
        assert [block for block, place in enumerate(book.table[b]) if place >= 0] == list(range(len(tokens) // 64))
    assert sorted({p for row in book.table for p in row if p >= 0}) == list(range(int(names["used"])))

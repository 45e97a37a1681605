"""GPU parity of the decoding operators against their plain 64-bit forms
(tests/decoding_reference.py), one by one and as a decoding step runs them."""

from __future__ import annotations

import math

import pytest
import torch

import decoding_reference as plain

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _rand(shape, seed, dtype, spread=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype)


def _near(got, want, bound, what):
    """|got - want| <= bound elementwise; NaN exactly where ``want`` has it."""

    got = got.double().cpu()
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    off = torch.where(torch.isnan(want), torch.zeros_like(want), (got - want).abs() - bound)
    assert float(off.max()) <= 0 if off.numel() else True, f"{what}: {float(off.max()):.3g} above the bound"


# ---------------------------------------------------------------------------
# norm and rotation


def _rotary_case(device, *, batch, seq, heads, kv_heads, dim, rotary, dtype, norm="rms", interleaved=False,
                 params=F32, bias=False, starts=None, rows=None, weights=True, seed=0):
    from solution.kernels.norm import hip_qk_norm_rotary, rotary_table

    # views of a packed projection's output, as a program has them
    packed = _rand((batch, seq, heads + 2 * kv_heads, dim), seed, dtype)
    wq, wk, bq, bk = (_rand((dim,), seed + i, params) if on else None
                      for i, on in ((1, weights), (2, weights), (3, bias), (4, bias)))
    most = max([0] if starts is None else starts) + seq
    table = rotary_table(most if rows is None else rows, rotary, device="cpu") if rotary else None
    starts_t = None if starts is None else torch.tensor(starts, dtype=torch.int32)
    to = lambda t: None if t is None else t.to(device)  # noqa: E731
    on_gpu = packed.to(device)
    with torch.inference_mode():
        got = hip_qk_norm_rotary(
            on_gpu[:, :, :heads].transpose(1, 2), on_gpu[:, :, heads : heads + kv_heads].transpose(1, 2),
            to(wq), to(wk), to(table), to(starts_t), query_bias=to(bq), key_bias=to(bk), norm=norm,
            interleaved=interleaved,
        )
    assert got[2] == "hip_qk_norm_rotary"
    for out, view, w, b in ((got[0], packed[:, :, :heads], wq, bq), (got[1], packed[:, :, heads : heads + kv_heads], wk, bk)):
        want = plain.norm_rotary(view.transpose(1, 2).double(), w, b, table, starts_t, norm=norm, eps=1e-6,
                                 interleaved=interleaved)
        # one rounding, and fp32 arithmetic on values of up to a row's largest: a sum of
        # `dim` squares, a square root and two products of two terms, (dim / 2 + 16) 2^-24
        size = want.nan_to_num().abs().amax(-1, keepdim=True) * 2 + 1
        bound = plain.half_step(dtype) * want.nan_to_num().abs() + (dim / 2 + 16) * 2.0**-24 * size
        assert out.is_contiguous() and out.dtype == dtype
        _near(out, want, bound, f"rotary batch={batch} seq={seq} dim={dim} {dtype}")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_types_and_head_dims(gpu_device, dtype, dim, interleaved):
    _rotary_case(gpu_device, batch=2, seq=5, heads=6, kv_heads=2, dim=dim, rotary=dim, dtype=dtype,
                 interleaved=interleaved, starts=[0, 999], seed=dim)


@pytest.mark.parametrize(
    "changes",
    [
        dict(heads=1, kv_heads=1, seq=1),
        dict(heads=16, kv_heads=16, seq=1),
        dict(heads=5, kv_heads=3, seq=67),
        dict(heads=40, kv_heads=5, seq=3),
        dict(batch=1, heads=12, kv_heads=4, seq=333, starts=[7]),
        dict(starts=None),
        dict(rotary=0),
        dict(rotary=0, norm="layer", bias=True),
        dict(rotary=32),
        dict(rotary=16, dim=128),
        dict(rotary=48),
        dict(rotary=24, interleaved=True),
        dict(norm="layer"),
        dict(norm="layer", bias=True, interleaved=True),
        dict(bias=True, params=BF16),
        dict(weights=False),
        # positions before and behind the table
        dict(starts=[-2, 20], rows=22, seq=4),
        dict(starts=[0, 5], rows=8, rotary=32, interleaved=True),
    ],
)
def test_rotary_layouts(gpu_device, changes):
    sizes = dict(batch=2, seq=4, heads=4, kv_heads=2, dim=64, rotary=64, dtype=BF16, starts=[0, 50], seed=9)
    _rotary_case(gpu_device, **{**sizes, **changes})


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rotary_of_many_tokens_is_that_of_few(gpu_device, dtype):
    """Outputs past the caches, several groups of heads a wave, and few tokens: the same bits."""

    from solution.kernels.norm import hip_qk_norm_rotary, rotary_table

    seq = 34_001 if dtype is BF16 else 17_001
    packed = torch.randn(2, seq, 20, 64, generator=torch.Generator(device=gpu_device).manual_seed(5), device=gpu_device).to(dtype)
    table = rotary_table(seq + 9, 64, device=gpu_device)
    weight = torch.linspace(0.5, 1.5, 64, device=gpu_device)
    views = lambda t: (t[:, :, :16].transpose(1, 2), t[:, :, 16:].transpose(1, 2))  # noqa: E731
    starts = lambda at: torch.tensor([at, at + 9], dtype=torch.int32, device=gpu_device)  # noqa: E731
    with torch.inference_mode():
        query, key, _ = hip_qk_norm_rotary(*views(packed), weight, weight, table, starts(0))
        assert query.numel() * query.element_size() > 128 << 20
        for at, count in ((0, 1), (17_000, 1), (4_999, 3_000), (seq - 77, 77)):
            part = hip_qk_norm_rotary(*views(packed[:, at : at + count]), weight, weight, table, starts(at))
            assert torch.equal(query[:, :, at : at + count], part[0]) and torch.equal(key[:, :, at : at + count], part[1])


def test_rotary_of_zeros_and_broadcast_heads(gpu_device):
    from solution.kernels.norm import hip_qk_norm_rotary, rotary_table

    table = rotary_table(8, 64, device=gpu_device)
    one = _rand((1, 1, 4, 64), 3, BF16).to(gpu_device)
    zeros = torch.zeros(3, 2, 4, 64, dtype=BF16, device=gpu_device)
    with torch.inference_mode():
        query, key, _ = hip_qk_norm_rotary(one.expand(3, 6, 4, 64), zeros, None, None, table)
    want = plain.norm_rotary(one.double().cpu(), None, None, table.cpu(), None, norm="rms", eps=1e-6, interleaved=False)
    _near(query, want.expand(3, 6, 4, 64), 2.0**-8 * want.abs() + 2.0**-17, "broadcast heads")
    assert bool((key == 0).all())


def test_rotary_refusals(gpu_device):
    from solution.kernels.norm import hip_qk_norm_rotary, rotary_table

    q, k = (torch.zeros(2, h, 4, 64, dtype=BF16, device=gpu_device) for h in (4, 2))
    w = torch.ones(64, device=gpu_device)
    table = rotary_table(8, 64, device=gpu_device)
    starts = torch.zeros(2, dtype=torch.int32, device=gpu_device)
    good = dict(query=q, key=k, query_weight=w, key_weight=w, table=table, starts=starts)
    hip_qk_norm_rotary(**good)
    for changes in (
        dict(query=q.double()), dict(key=k.half()), dict(key=k[:1]), dict(query=q[..., :32], key=k[..., :32]),
        dict(query=q.transpose(2, 3)), dict(query_weight=w[:32]), dict(key_weight=w.half()), dict(starts=starts.long()),
        dict(starts=starts[:1]), dict(table=table.half()), dict(table=table[:, :40].contiguous()), dict(table=table.t()),
        dict(table=table.cpu()), dict(norm="batch"), dict(eps=-1.0), dict(query=q[0]),
        dict(query=q.clone().requires_grad_()), dict(query_weight=w.clone().requires_grad_()),
    ):
        with pytest.raises(RuntimeError, match="ineligible"):
            hip_qk_norm_rotary(**{**good, **changes})


# ---------------------------------------------------------------------------
# the cache


class _Tokens:
    """Sequences' keys and values as the program appends them, and the cache beside."""

    def __init__(self, device, lengths, kv_heads, dim, dtype, *, room=None, seed=0, spread=1.0, spare=3):
        from solution.kernels.attention import BlockCache

        self.device, self.dtype, self.lengths = device, dtype, list(lengths)
        batch, most = len(lengths), max(list(lengths) + [1])
        room = most if room is None else room
        width = room // 64 + 1
        order = torch.randperm(batch * width + spare, generator=torch.Generator().manual_seed(seed + 5))
        table = order[: batch * width].to(torch.int32).reshape(batch, width)
        self.key = _rand((batch, kv_heads, most, dim), seed, dtype, spread)
        self.value = _rand((batch, kv_heads, most, dim), seed + 1, dtype, spread)
        self.cache = BlockCache.allocate(batch, kv_heads, dim, max_tokens=room, num_blocks=batch * width + spare,
                                         dtype=dtype, device=device, block_table=table.to(device))

    def append(self, starts, counts, padded=None):
        """Append tokens starts[b] .. starts[b] + counts[b] - 1 of each sequence."""

        from solution.kernels.attention import hip_block_cache_append

        seq = padded or max(max(counts), 1)
        batch, heads, _, dim = self.key.shape
        # rows of a packed projection; what stands behind the counts is not to be read
        packed = torch.full((batch, seq, 2 * heads, dim), math.nan, dtype=self.dtype)
        for b, (start, count) in enumerate(zip(starts, counts)):
            packed[b, :count, :heads] = self.key[b, :, start : start + count].transpose(0, 1)
            packed[b, :count, heads:] = self.value[b, :, start : start + count].transpose(0, 1)
        packed = packed.to(self.device)
        to = lambda v: torch.tensor(v, dtype=torch.int32, device=self.device)  # noqa: E731
        with torch.inference_mode():
            marker = hip_block_cache_append(
                self.cache, packed[:, :, :heads].transpose(1, 2), packed[:, :, heads:].transpose(1, 2), to(starts),
                None if counts == [seq] * batch else to(counts),
            )
        assert marker == "hip_block_cache_append"

    def fill(self):
        self.append([0] * len(self.lengths), self.lengths)
        return self

    def stored(self, b, h, length=None):
        length = self.lengths[b] if length is None else length
        return plain.stored_tokens(self.key[b, h, :length].double(), self.value[b, h, :length].double())

    def read(self, firsts, lengths, tokens):
        from solution.kernels.attention import hip_block_cache_read

        to = lambda v: torch.tensor(v, dtype=torch.int32, device=self.device)  # noqa: E731
        with torch.inference_mode():
            key, value, marker = hip_block_cache_read(self.cache, to(firsts), to(lengths), tokens)
        assert marker == "hip_block_cache_read"
        return key.double().cpu(), value.double().cpu()

    def check(self, lengths=None):
        """Everything that the cache holds is what the plain form stores."""

        lengths = self.lengths if lengths is None else lengths
        batch, heads, _, dim = self.key.shape
        key, value = self.read([0] * batch, lengths, max(lengths) + 3)
        for b in range(batch):
            for h in range(heads):
                want_key, want_value = self.stored(b, h, lengths[b])
                n = lengths[b]
                assert torch.equal(value[b, h, :n], want_value), (b, h)
                assert torch.equal(key[b, h, :n].nan_to_num(7e4), want_key.nan_to_num(7e4)), (b, h)
                assert not bool(key[b, h, n:].any()) and not bool(value[b, h, n:].any())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths", [[1], [63], [64], [65], [1, 0, 64, 129, 300, 127]])
def test_append_stores_what_the_plain_form_stores(gpu_device, lengths, dtype, dim):
    _Tokens(gpu_device, lengths, 3, dim, dtype, seed=len(lengths)).fill().check()


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 128)])
def test_cache_does_not_depend_on_the_steps(gpu_device, dtype, dim):
    whole = _Tokens(gpu_device, [300, 193, 70], 2, dim, dtype, seed=4).fill()
    steps = _Tokens(gpu_device, [300, 193, 70], 2, dim, dtype, seed=4)
    held = [0, 0, 0]
    for chunk in ([1, 1, 1], [62, 0, 64], [1, 130, 0], [1, 1, 5], [64, 1, 0], [150, 0, 0], [1, 60, 0], [20, 0, 0]):
        steps.append(held, chunk, padded=max(chunk) + 2)
        held = [a + b for a, b in zip(held, chunk)]
        steps.check(held)
    assert held == [300, 193, 70]
    for name in ("key_codes", "value_codes", "key_scales", "value_scales"):
        assert torch.equal(getattr(whole.cache, name), getattr(steps.cache, name)), name
    for b, length in enumerate(held):  # tails up to the last token
        n = length % 64
        assert torch.equal(whole.cache.key_tail[b, :, :n], steps.cache.key_tail[b, :, :n])
        assert torch.equal(whole.cache.value_tail[b, ..., :n], steps.cache.value_tail[b, ..., :n])


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 64), (BF16, 128)])
def test_appends_of_few_and_several_tokens(gpu_device, dtype, dim):
    """Within a block, up to its end, over it and over several, a few tokens and many."""

    steps = [(5, 8), (20, 7), (9, 1), (30, 47), (1, 2), (64, 63), (7, 1), (100, 9), (8, 70), (0, 3), (63, 8), (13, 64)]
    lengths = [sum(s[b] for s in steps) for b in range(2)]
    t = _Tokens(gpu_device, lengths, 2, dim, dtype, seed=261)
    t.key[0, 1, 24, 3], t.value[1, 0, 14, 5] = math.inf, math.nan
    held = [0, 0]
    for step in steps:
        t.append(held, list(step))
        held = [a + b for a, b in zip(held, step)]
        t.check(held)


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F16, 128)])
def test_tokens_taken_back(gpu_device, dtype, dim):
    """Within the incomplete block, to a multiple of 64, and elsewhere by way of the read:
    the cache then holds what it would without the tokens that were taken back."""

    t = _Tokens(gpu_device, [200, 200, 130], 2, dim, dtype, seed=321)
    t.append([0, 0, 0], [200, 200, 130])
    held = [195, 64, 128]  # the second goes back to a border two blocks below, the third to its own block's first token
    fresh = _rand((3, 2, 200, dim), 322, dtype)
    for b, n in enumerate(held):
        t.key[b, :, n:] = fresh[b, :, n:]
        t.value[b, :, n:] = -fresh[b, :, n:]
    t.check(held)
    t.append(held, [3, 70, 1])
    held = [198, 134, 129]
    t.check(held)
    _check_attention(t, _rand((3, 4, 1, dim), 323, dtype), [n - 1 for n in held], [1, 1, 1])
    # back to 100 of the first sequence's tokens: its second block's first 36 are coded ones by now
    key, value = t.read([64, 0, 0], held, 36)
    t.key[0, :, 64:100], t.value[0, :, 64:100] = key[0].to(dtype), value[0].to(dtype)
    t.append([64, 134, 129], [36, 0, 0])
    t.check([100, 134, 129])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scales_of_extreme_blocks(gpu_device, dtype):
    t = _Tokens(gpu_device, [64 * 6 + 1], 1, 64, dtype, seed=11)
    most = torch.finfo(dtype).max
    t.key[0, 0, :64] = 0.0  # a block of zeros
    t.key[0, 0, 64:128] *= 1e-4
    t.key[0, 0, 130, 3] = 448.0  # on the border of a scale, and just above it
    t.key[0, 0, 128:192] = t.key[0, 0, 128:192].clamp(-448, 448)
    t.key[0, 0, 195, 7] = 450.0 if dtype is BF16 else 448.25
    t.value[0, 0, :64] = torch.finfo(dtype).smallest_normal
    t.value[0, 0, 64:128, 5] = most / 2
    t.value[0, 0, 256:320] = 2.0**-24 if dtype is F16 else 2.0**-133
    t.fill()
    scales = t.cache.key_scales.cpu()[t.cache.block_table.cpu()[0, :6].long(), 0]
    assert scales[0] == 1.0 and scales[2] == 1.0 and scales[3] == 2.0
    t.check()
    # the largest value of the type: its code times the scale leaves the type's range, and is read as the largest
    t = _Tokens(gpu_device, [64], 1, 64, dtype, seed=12)
    t.value[0, 0, 9, 9] = most
    t.fill()
    _, value = t.read([0], [64], 64)
    assert value[0, 0, 9, 9] == most


def test_non_finite_tokens_are_kept_apart(gpu_device):
    t = _Tokens(gpu_device, [200, 130], 2, 64, BF16, seed=21)
    t.key[0, 1, 5, 3] = math.nan
    t.key[0, 0, 70, 0] = math.inf
    t.value[0, 0, 71, 63] = -math.inf
    t.value[1, 1, 129, 1] = math.nan  # in the tail
    t.key[1, 0, 128] = math.nan
    t.fill().check()
    # the same token by token around the border of a block: a tail's NaN is coded later
    t2 = _Tokens(gpu_device, [200, 130], 2, 64, BF16, seed=21)
    t2.key, t2.value = t.key, t.value
    t2.append([0, 0], [63, 127])
    t2.append([63, 127], [10, 2])
    t2.append([73, 129], [127, 1])
    t2.check()


def test_read_of_any_span(gpu_device):
    t = _Tokens(gpu_device, [200, 130, 0], 2, 64, F16, seed=31).fill()
    whole = [torch.stack([t.stored(b, h)[i].nan_to_num() if t.lengths[b] else torch.zeros(0, 64).double()
                          for b in range(1) for h in range(2)]) for i in range(2)]
    for firsts, tokens in (([0, 0, 0], 0), ([63, 1, 0], 1), ([70, 129, 5], 90), ([-5, -70, -1], 100), ([199, 500, 64], 70)):
        got = t.read(firsts, t.lengths, tokens)
        for i in range(2):
            assert got[i].shape == (3, 2, tokens, 64)
            for row in range(tokens):
                p = firsts[0] + row
                want = whole[i][:, p] if 0 <= p < 200 else torch.zeros(2, 64).double()
                assert torch.equal(got[i][0, :, row], want), (firsts, row)
            assert not bool(got[i][2].any())


def test_pages_outside_the_cache(gpu_device):
    from solution.kernels.attention import hip_block_cache_attention

    t = _Tokens(gpu_device, [300, 300, 300], 2, 64, BF16, seed=41)
    codes = t.cache.key_codes.clone()
    t.cache.block_table[0, 1] = t.cache.key_codes.shape[0]
    t.cache.block_table[1, 3] = -1
    t.fill()
    key, value = t.read([0] * 3, [300] * 3, 300)
    lost = torch.zeros(3, 300, dtype=torch.bool)
    lost[0, 64:128] = lost[1, 192:256] = True
    assert bool((key.isnan().all(-1) == lost[:, None]).all()) and bool((value.isnan().all(-1) == lost[:, None]).all())
    named = t.cache.block_table[t.cache.block_table.ge(0) & t.cache.block_table.lt(codes.shape[0])].long()
    others = torch.ones(codes.shape[0], dtype=torch.bool, device=gpu_device)
    others[named] = False
    assert torch.equal(t.cache.key_codes[others], codes[others])
    # rows before the lost page answer, rows that see it are NaN
    query = _rand((3, 4, 130, 64), 42, BF16).to(gpu_device)
    starts = torch.tensor([0, 150, 170], dtype=torch.int32, device=gpu_device)
    with torch.inference_mode():
        out = hip_block_cache_attention(query, t.cache, starts)[0].cpu()
    bad = out.isnan().all(-1)
    assert bool(out.isnan().any(-1).eq(bad).all())
    position = starts.cpu()[:, None] + torch.arange(130)
    first_lost = torch.tensor([64, 192, 10**6])[:, None]
    assert torch.equal(bad, position >= first_lost)


def test_lengths_beyond_the_table_and_sequences_without_tokens(gpu_device):
    from solution.kernels.attention import hip_block_cache_append, hip_block_cache_attention

    t = _Tokens(gpu_device, [100, 100, 100], 2, 64, BF16, room=127, seed=51).fill()
    assert t.cache.block_table.shape[1] == 2
    before = {n: getattr(t.cache, n).clone() for n in ("key_codes", "value_codes", "key_tail", "value_tail", "key_scales")}
    kv = _rand((3, 2, 2, 64), 52, BF16).to(gpu_device)
    starts = torch.tensor([-1, 100, 2**31 - 1], dtype=torch.int32, device=gpu_device)
    counts = torch.tensor([2, -3, 0], dtype=torch.int32, device=gpu_device)
    with torch.inference_mode():
        hip_block_cache_append(t.cache, kv, kv, starts, counts)
        for name, want in before.items():
            assert torch.equal(getattr(t.cache, name), want), name
        query = _rand((3, 4, 2, 64), 53, BF16).to(gpu_device)
        out = hip_block_cache_attention(query, t.cache, starts, counts)[0]
        assert not bool(out.any())
        # more tokens than the table has room for: NaN, and an end
        far = torch.tensor([192, 2**31 - 64, 98], dtype=torch.int32, device=gpu_device)
        out = hip_block_cache_attention(query, t.cache, far)[0].cpu()
    assert bool(out[:2].isnan().all()) and bool(out[2].isfinite().all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,seq", [(2, 170), (8, 150), (2, 70), (16, 66)])
def test_rows_before_the_end_of_the_table_answer(gpu_device, heads, seq, dim):
    """A chunk that passes the table's room: rows that see only blocks with a place answer, the others are NaN."""

    starts = [127, 100, 0, 64, 128, 150]
    counts = [seq, max(seq - 10, 92), seq, 0, 64, seq]
    counts = [min(c, seq) for c in counts]
    t = _Tokens(gpu_device, [s + c for s, c in zip(starts, counts)], 2, dim, BF16, room=127, seed=291)
    assert t.cache.block_table.shape[1] == 2
    t.append(starts=[0] * 6, counts=starts)
    t.append(starts, counts)
    query = _rand((6, heads, seq, dim), 292, BF16)
    out = _attend(t, query, starts, counts)
    for b, (start, count) in enumerate(zip(starts, counts)):
        lost = (start + torch.arange(seq) >= 128) & (torch.arange(seq) < count) & (start + count >= 192)
        assert bool(out[b].isnan().all(-1).eq(lost).all()) and bool(out[b].isnan().any(-1).eq(lost).all()), b
        seen = [i for i in (0, 1, 27, 28, 63, 64, 127) if i < count and not lost[i]]
        for h in range(heads):
            keys, values = t.stored(b, h // (heads // 2), start + count)
            for i in seen:
                q = query[b, h, i].double()
                want, size = plain.attention(q, keys, values, start + i, dim**-0.5)
                bound = plain.attention_bound(want, size, q, keys, start + i, dim**-0.5, BF16)
                _near(out[b, i].reshape(heads, dim)[h], want, bound, f"sequence {b} head {h} row {i}")


# ---------------------------------------------------------------------------
# attention over the cache


def _attend(t, query, starts, counts=None, **options):
    from solution.kernels.attention import hip_block_cache_attention

    to = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32, device=t.device)  # noqa: E731
    with torch.inference_mode():
        out, marker = hip_block_cache_attention(query.to(t.device), t.cache, to(starts), to(counts), **options)
    assert marker == "hip_block_cache_attention"
    return out.cpu()


def _check_attention(t, query, starts, counts=None, *, scale=None, rows=None, **options):
    """Every row (or the rows named) against the plain form over what the cache stands for."""

    batch, heads, seq, dim = query.shape
    group = heads // t.key.shape[1]
    out = _attend(t, query, starts, counts, scale=scale, **options)
    assert out.shape == (batch, seq, heads * dim) and out.dtype == t.dtype
    out = out.reshape(batch, seq, heads, dim)
    scale = dim**-0.5 if scale is None else scale
    for b in range(batch):
        count = seq if counts is None else counts[b]
        assert not bool(out[b, count:].any())
        for h in range(heads):
            keys, values = t.stored(b, h // group, starts[b] + count)
            for i in range(count) if rows is None else [r for r in rows if r < count]:
                q = query[b, h, i].double()
                want, size = plain.attention(q, keys, values, starts[b] + i, scale)
                bound = plain.attention_bound(want, size, q, keys, starts[b] + i, scale, t.dtype)
                _near(out[b, i, h], want, bound, f"attention sequence {b} head {h} row {i} of {starts[b]}+{count}")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2), (12, 1), (20, 1), (6, 2)])
def test_one_token_over_ragged_histories(gpu_device, heads, kv_heads, dtype, dim):
    lengths = [1, 2, 63, 64, 65, 128, 129, 500, 1100]
    t = _Tokens(gpu_device, lengths, kv_heads, dim, dtype, seed=heads + dim).fill()
    query = _rand((len(lengths), heads, 1, dim), 61, dtype)
    _check_attention(t, query, [n - 1 for n in lengths])


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(4, 4, 64, BF16), (8, 2, 64, F16), (4, 1, 128, BF16), (3, 3, 128, F16)])
@pytest.mark.parametrize("seq", [2, 5, 17, 33, 64, 70, 150])
def test_chunks_over_ragged_histories(gpu_device, seq, heads, kv_heads, dim, dtype):
    counts = [seq, 1, max(1, seq // 2), 0, seq]
    starts = [0, 130, 61, 40, 700]
    t = _Tokens(gpu_device, [a + b for a, b in zip(starts, counts)], kv_heads, dim, dtype, seed=seq).fill()
    query = _rand((5, heads, seq, dim), 71, dtype)
    rows = None if seq <= 17 else [0, 1, 2, 3, 15, 16, 31, 32, 47, 63, 64, 69, 100, seq - 1]
    _check_attention(t, query, starts, counts, rows=rows)


@pytest.mark.parametrize("batch,seq", [(20, 100), (64, 100), (64, 40)])
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, BF16), (64, F16)])
def test_chunks_of_many_rows_over_short_histories(gpu_device, batch, seq, dim, dtype):
    """Rows that fill the card: one or two waves share a row's tokens."""

    starts = [(37 * b) % 131 for b in range(batch)]
    counts = [seq if b % 3 else (b * 7) % (seq + 1) for b in range(batch)]
    t = _Tokens(gpu_device, [a + b for a, b in zip(starts, counts)], 8, dim, dtype, seed=251).fill()
    _check_attention(t, _rand((batch, 8, seq, dim), 252, dtype), starts, counts, rows=[0, 31, 39, 57, 99])


@pytest.mark.parametrize("max_length", [None, 1, 500, 5000])
@pytest.mark.parametrize("seq", [1, 20, 80])
def test_long_histories_in_parts(gpu_device, seq, max_length):
    starts = [4990 - seq, 63, 2500, 0]
    t = _Tokens(gpu_device, [s + seq for s in starts], 1, 64, BF16, room=6000, seed=81).fill()
    query = _rand((4, 2, seq, 64), 82, BF16)
    _check_attention(t, query, starts, rows=[0, 7, seq - 1], max_length=max_length)


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (64, F16), (128, BF16), (128, F16)])
@pytest.mark.parametrize("seq", [1, 20, 80, 150])
def test_parts_of_every_type_and_head_dim(gpu_device, seq, dim, dtype):
    """More than one part a row and their merge, in each kernel, beyond 8192 tokens and before."""

    from solution.kernels.hip import load_library

    starts, counts = [12_000 - seq, 63, 2_500, 0], [seq, seq, max(1, seq // 2), 1]
    t = _Tokens(gpu_device, [s + c for s, c in zip(starts, counts)], 1, dim, dtype, room=12_500, seed=301).fill()
    query = _rand((4, 2, seq, dim), 302, dtype)
    for max_length in (None, 4_000):
        most = t.cache.max_tokens if max_length is None else max_length
        parts = load_library().sah_block_cache_attention_workspace_bytes(4, seq, 2, 1, dim, most) // (4 * seq * 2 * (dim + 2) * 4)
        assert parts > 1
        _check_attention(t, query, starts, counts, rows=[0, 7, 33, seq - 1], max_length=max_length)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,seq", [(64, 1), (4, 8), (2, 150)])
def test_values_all_alike_come_back_exactly(gpu_device, heads, seq, dtype, dim):
    """The weights that the values take are those that the row's sum adds up.  1.875 is a
    code of every block scale; half a step of fp16 there is 2.6e-4 of it, the rounding of
    a weight to fp16 up to 4.9e-4."""

    lengths = [3000 + 37 * b for b in range(8)]
    t = _Tokens(gpu_device, lengths, 1, dim, dtype, seed=311)
    t.value[:] = 1.875
    t.fill()
    query = _rand((8, heads, seq, dim), 312, dtype)
    for scale in (0.25, 1.0, 2.0):
        out = _attend(t, query, [n - seq for n in lengths], scale=scale, max_length=1)
        assert bool((out == 1.875).all()), scale


@pytest.mark.parametrize("scale", [0.5, -0.125, 0.0, 1e-30, 3.0])
@pytest.mark.parametrize("seq", [1, 40])
def test_scales_of_the_scores(gpu_device, scale, seq):
    t = _Tokens(gpu_device, [seq + 100, seq + 3], 2, 64, BF16, seed=91).fill()
    _check_attention(t, _rand((2, 4, seq, 64), 92, BF16), [100, 3], scale=scale)


def test_blocks_of_very_different_sizes(gpu_device):
    t = _Tokens(gpu_device, [64 * 5 + 10], 1, 64, BF16, seed=95)
    for block, size in enumerate((1e-30, 1e20, 1e-6, 0.0, 1e30)):
        t.value[0, 0, 64 * block : 64 * block + 64] *= size
    t.key[0, 0, 64:128] *= 30.0
    t.key[0, 0, 256:320] = 0.0
    t.fill()
    _check_attention(t, _rand((1, 8, 1, 64), 96, BF16), [t.lengths[0] - 1])
    _check_attention(t, _rand((1, 3, 329, 64), 97, BF16), [0], [329], rows=[0, 63, 64, 127, 200, 255, 256, 328])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,start,seq", [(1, 13, 150), (3, 5, 140), (2, 50, 90), (1, 40, 300)])
def test_later_blocks_leave_earlier_rows_alone(gpu_device, heads, start, seq, dim):
    """Value scales more than 2^126 apart, rows of one wave on both sides of a block's
    border, and 16 blocks before it, so that every wave has met the small values."""

    border, start = 64 * 17, 64 * 16 + start
    t = _Tokens(gpu_device, [start + seq], 1, dim, BF16, seed=271)
    t.value[0, 0, :border] *= 1e-20
    t.value[0, 0, border:] *= 1e30
    t.fill()
    query = _rand((1, heads, seq, dim), 272, BF16)
    last = border - 1 - start
    rows = [0, last - 2, last - 1, last, last + 1, last + 2, seq - 1]
    _check_attention(t, query, [start], rows=rows, max_length=1)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,seq", [(1, 1), (6, 2), (1, 150), (3, 120)])
@pytest.mark.parametrize("last", [64 * 27, 64 * 27 + 9])
def test_blocks_without_weight_leave_small_outputs_alone(gpu_device, last, heads, seq, dim):
    """A row whose weights of a block are all zero answers from the others, whatever the block holds."""

    t = _Tokens(gpu_device, [last], 1, dim, BF16, seed=281)
    near = 64 * 17  # the tokens before it have all the weight
    t.key[0, 0] = (t.key[0, 0].float() * 0.25 + 8.0).to(BF16)
    t.key[0, 0, near:] = (t.key[0, 0, near:].float() - 16.0).to(BF16)  # scores some 16 dim^0.5 below
    t.value[0, 0, :near] *= 1e-20
    t.value[0, 0, near:] *= 1e30
    t.fill()
    query = (torch.ones(1, heads, seq, dim) + 0.1 * _rand((1, heads, seq, dim), 282, F32)).to(BF16)
    start = last - seq
    out = _attend(t, query, [start], max_length=1).reshape(seq, heads, dim)
    keys, values = t.stored(0, 0)
    for h in range(heads):
        for i in {0, seq // 2, seq - 1}:
            q = query[0, h, i].double()
            scores = keys[: start + i + 1] @ q * dim**-0.5
            assert float(scores[:near].max() - scores[near:].max()) > 100.0  # weights below 2^-144
            weights = torch.softmax(scores[:near], 0)
            want, sizes = weights @ values[:near], weights @ values[:near].abs()
            inner = 2 * (2.0**-11 + 2 * (dim + 4) * 2.0**-24 * float((keys[:near].abs() @ q.abs()).max()) * dim**-0.5 + 2.0**-20)
            _near(out[i, h], want, 2.0**-8 * want.abs() + (1 + 2.0**-8) * inner * sizes, f"head {h} row {i}")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,seq,max_length", [(1, 1, None), (2, 150, None), (1, 1, 1), (2, 150, 1)])
def test_the_types_largest_values(gpu_device, heads, seq, max_length, dtype):
    """Their codes stand for more than the type holds; the answer stays in its range."""

    most = torch.finfo(dtype).max
    t = _Tokens(gpu_device, [6000], 1, 64, dtype, seed=341)
    t.value[..., :32], t.value[..., 32:] = most, -most
    t.fill()
    out = _attend(t, _rand((1, heads, seq, 64), 342, dtype), [6000 - seq], max_length=max_length).reshape(seq, heads, 64)
    # rounding of a code up (by 2^-4 at most) and back, and of weights; the tail holds the values themselves
    assert bool((out[..., :32] >= most * (1 - 2.0**-7)).all()) and bool((out[..., 32:] <= -most * (1 - 2.0**-7)).all())
    assert bool(out.isfinite().all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seq", [1, 150])
@pytest.mark.parametrize("size", [1e36, 1e-30])
def test_large_and_small_values_in_parts(gpu_device, size, seq, dim):
    """Parts are merged by their shares: outputs far from 1 neither overflow nor lose bits."""

    t = _Tokens(gpu_device, [9000, 5000], 1, dim, BF16, seed=351)
    t.value *= size
    t.fill()
    _check_attention(t, _rand((2, 2, seq, dim), 352, BF16), [9000 - seq, 5000 - seq], rows=[0, seq - 1])


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (64, F16), (128, BF16)])
@pytest.mark.parametrize("seq", [1, 5, 40])
def test_scores_that_grow_and_fall_along_the_history(gpu_device, seq, dim, dtype):
    """Every block's largest scores far above all before it, then far below."""

    sizes = (0.25, 1.0, 3.0, 8.0, 20.0, 40.0, 1.0, 0.1, 60.0, 2.0)
    length = 64 * len(sizes) * 5 + 7
    t = _Tokens(gpu_device, [length, length - 70], 1, dim, dtype, seed=241)
    for block in range(length // 64):
        t.key[:, :, 64 * block : 64 * block + 64] *= sizes[block // 5]
    t.fill()
    _check_attention(t, _rand((2, 4, seq, dim), 242, dtype), [length - seq, length - 70 - seq], rows=[0, seq - 1], max_length=1)


def test_strided_queries_and_broadcast_heads(gpu_device):
    from solution.kernels.attention import hip_block_cache_attention

    t = _Tokens(gpu_device, [150, 90], 2, 64, BF16, seed=101).fill()
    packed = _rand((2, 3, 10, 64), 102, BF16)
    _check_attention(t, packed[:, :, 1:7].transpose(1, 2), [147, 87])
    wide = packed.to(gpu_device)[:, :, 1:7].transpose(1, 2)
    assert not wide.is_contiguous()
    starts = torch.tensor([147, 87], dtype=torch.int32, device=gpu_device)
    with torch.inference_mode():
        assert torch.equal(hip_block_cache_attention(wide, t.cache, starts)[0],
                           hip_block_cache_attention(wide.contiguous(), t.cache, starts)[0])
        one = wide[:, :1].expand(2, 6, 3, 64)
        assert torch.equal(hip_block_cache_attention(one, t.cache, starts)[0],
                           hip_block_cache_attention(one.contiguous(), t.cache, starts)[0])


@pytest.mark.parametrize("seq", [1, 30])
def test_non_finite_tokens_touch_only_the_rows_that_see_them(gpu_device, seq):
    length = 200
    for place in (length - 1, length - 20, 70):
        clean = _Tokens(gpu_device, [length], 2, 64, BF16, seed=111)
        bad = _Tokens(gpu_device, [length], 2, 64, BF16, seed=111)
        for t in (clean, bad):  # the same coded blocks: the token takes no part in a scale
            t.key[0, 0, place] = t.value[0, 0, place] = 0.0
        bad.value[0, 0, place, 3] = math.nan
        query = _rand((1, 4, seq, 64), 112, BF16)
        start = length - seq
        want, got = (_attend(t.fill(), query, [start]).reshape(seq, 4, 64) for t in (clean, bad))
        sees = torch.arange(start, length) >= place
        assert bool(got[sees][:, :2].isnan().all())
        assert torch.equal(got[~sees], want[~sees]) and torch.equal(got[:, 2:], want[:, 2:])


def test_what_stands_behind_the_last_token_is_not_read(gpu_device):
    t = _Tokens(gpu_device, [70, 64], 2, 64, BF16, seed=121).fill()
    query = _rand((2, 4, 1, 64), 122, BF16)
    want = _attend(t, query, [69, 63])
    t.cache.key_tail[0, :, 6:] = math.nan
    t.cache.value_tail[0, ..., 6:] = math.nan
    t.cache.key_tail[1] = math.nan
    t.cache.value_tail[1] = math.nan
    spare = torch.ones(t.cache.key_codes.shape[0], dtype=torch.bool, device=gpu_device)
    spare[t.cache.block_table[:, 0].long()] = False
    t.cache.key_codes[spare] = 0x7F
    t.cache.value_codes[spare] = 0x7F
    t.cache.block_table[:, 1:] = -1
    assert torch.equal(_attend(t, query, [69, 63]), want)


def test_blocks_shared_by_sequences(gpu_device):
    """A common beginning is held once: the second sequence's table names the first's blocks."""

    t = _Tokens(gpu_device, [200, 192], 2, 64, F16, seed=131)
    t.key[1, :, :192], t.value[1, :, :192] = t.key[0, :, :192], t.value[0, :, :192]
    t.append([0, 0], [200, 0])
    t.cache.block_table[1, :3] = t.cache.block_table[0, :3]
    query = _rand((1, 4, 1, 64), 132, F16).expand(2, 4, 1, 64)
    # the second holds the 192 tokens of the blocks, and asks from the last of them
    _check_attention(t, query.contiguous(), [199, 191])


def test_cache_of_more_than_four_gigabytes(gpu_device):
    from solution.kernels.attention import BlockCache

    t = _Tokens(gpu_device, [130, 70], 16, 64, BF16, seed=141)
    blocks = 70_001  # 64 KiB of codes each, for keys and for values
    table = torch.tensor([[70_000, 65_537, 3], [66_000, 0, 32_768]], dtype=torch.int32, device=gpu_device)
    t.cache = BlockCache.allocate(2, 16, 64, max_tokens=200, num_blocks=blocks, dtype=BF16, device=gpu_device, block_table=table)
    t.fill().check()
    _check_attention(t, _rand((2, 16, 1, 64), 142, BF16), [129, 69])


@pytest.mark.parametrize("dim,dtype", [(64, BF16), (64, F16), (128, F16), (128, BF16)])
@pytest.mark.parametrize("seq", [1, 9, 40])
def test_more_blocks_than_one_look_up_of_a_wave(gpu_device, seq, dim, dtype):
    """Histories far beyond max_length: every wave's blocks come in more than one look-up of 64."""

    starts = [36_000, 9_000 if seq == 1 else 17_500]
    t = _Tokens(gpu_device, [s + seq for s in starts], 1, dim, dtype, seed=211).fill()
    query = _rand((2, 2, seq, dim), 212, dtype)
    _check_attention(t, query, starts, rows=[0, seq - 1], max_length=1)
    if seq == 1:
        return
    # a page outside the cache in the second look-up, which every row sees
    t.cache.block_table[0, 550] = -1
    t.cache.block_table[1, 265] = t.cache.key_codes.shape[0]
    assert bool(_attend(t, query, starts, max_length=1).isnan().all())


def test_many_look_ups_in_parts(gpu_device):
    """Four waves a workgroup and several parts, with more than 64 blocks a wave; and
    more than 64 parts."""

    t = _Tokens(gpu_device, [150_000], 1, 64, BF16, seed=215).fill()
    query = _rand((1, 2, 1, 64), 216, BF16)
    _check_attention(t, query, [149_999], max_length=8_300)
    _check_attention(t, query, [149_999])
    t.cache.block_table[0, 2_330] = -1
    assert bool(_attend(t, query, [149_999], max_length=8_300).isnan().all())


def test_more_rows_than_a_merge_takes(gpu_device):
    """2^26 padded rows and more, of which few have a query: the others are zeros."""

    batch, heads, seq, counts = 8, 64, 131_080, [5, 0, 70, 1, 33, 2, 64, 9]
    t = _Tokens(gpu_device, [100 + c for c in counts], 8, 64, BF16, seed=331).fill()
    query = _rand((batch, heads, 70, 64), 332, BF16)
    padded = torch.empty((batch, seq, heads, 64), dtype=BF16, device=gpu_device).transpose(1, 2)
    padded[:, :, :70] = query.to(gpu_device)
    starts, lengths = (torch.tensor(v, dtype=torch.int32, device=gpu_device) for v in ([100] * batch, counts))
    from solution.kernels.attention import hip_block_cache_attention

    with torch.inference_mode():
        out = hip_block_cache_attention(padded, t.cache, starts, lengths)[0]
        few = hip_block_cache_attention(query.to(gpu_device), t.cache, starts, lengths)[0]
    assert out.shape == (batch, seq, heads * 64) and not bool(out[:, 70:].any())
    for b, count in enumerate(counts):
        assert not bool(out[b, count:].any())
        for i in range(count):  # the same rows, the tokens split otherwise
            want = few[b, i].double()
            # two roundings of the output, and of weights (2^-11 each) on values of about 1
            assert float(((out[b, i].double() - want).abs() - 2.0**-7 * want.abs()).max()) <= 2.0**-9


@pytest.mark.parametrize("heads", [40, 96])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_query_heads_a_key_head(gpu_device, heads, dim):
    lengths = [1, 63, 64, 700]
    t = _Tokens(gpu_device, lengths, 1, dim, BF16, seed=heads).fill()
    _check_attention(t, _rand((4, heads, 1, dim), 213, BF16), [n - 1 for n in lengths])


@pytest.mark.parametrize("seq", [1, 3, 40])
def test_padded_rows_are_not_read(gpu_device, seq):
    """Queries behind the counts may hold anything; their outputs are zeros."""

    starts, counts = [70, 20, 300, 64], [seq, 0, max(1, seq // 2), 1]
    t = _Tokens(gpu_device, [a + b for a, b in zip(starts, counts)], 2, 64, BF16, seed=221).fill()
    query = _rand((4, 8, seq, 64), 222, BF16)
    for b, count in enumerate(counts):
        query[b, :, count:] = math.nan
    _check_attention(t, query, starts, counts, rows=[0, 1, seq - 1])


@pytest.mark.parametrize("width", [0, 2])
@pytest.mark.parametrize("dim", [64, 128])
def test_caches_without_blocks(gpu_device, dim, width):
    """Up to 63 tokens need no block; complete blocks have no place, and who sees one gets NaN."""

    from solution.kernels.attention import BlockCache, hip_block_cache_append

    t = _Tokens(gpu_device, [63, 17, 1], 2, dim, BF16, seed=231)
    table = torch.full((3, width), 0, dtype=torch.int32, device=gpu_device)
    t.cache = BlockCache.allocate(3, 2, dim, max_tokens=63, num_blocks=0, dtype=BF16, device=gpu_device, block_table=table)
    assert t.cache.max_tokens == 63 + 64 * width
    t.append([0] * 3, [40, 17, 1])
    t.append([40, 17, 1], [23, 0, 0])
    t.check()
    for seq in (1, 17):
        _check_attention(t, _rand((3, 8, seq, dim), 232, BF16), [63 - seq, max(0, 17 - seq), 0], [seq, seq, 1])
    kv = torch.ones((3, 2, 5, dim), dtype=BF16, device=gpu_device)
    starts = torch.tensor([63, 17, 1], dtype=torch.int32, device=gpu_device)
    with torch.inference_mode():
        hip_block_cache_append(t.cache, kv, kv, starts)
    for seq in (1, 5, 20):
        first = max(0, 22 - seq)
        query = _rand((3, 8, seq, dim), 233, BF16)
        out = _attend(t, query, [68 - seq, first, 0], [seq, min(seq, 22), min(seq, 6)])
        # the block of the first 64 tokens, which is lost, is seen by every row of the first sequence
        assert bool(out[0].isnan().all()) and not bool(out[1:].isnan().any())
    key, value = t.read([60, 0, 0], [68, 22, 6], 8)
    assert bool(key[0, :, :4].isnan().all()) and bool(value[0, :, :4].isnan().all())
    assert not bool(key[0, :, 4:].isnan().any()) and not bool(key[1:].isnan().any())


def test_attention_refusals(gpu_device):
    from solution.kernels.attention import hip_block_cache_append, hip_block_cache_attention, hip_block_cache_read

    t = _Tokens(gpu_device, [70, 64], 2, 64, BF16, seed=151).fill()
    q = torch.zeros(2, 4, 1, 64, dtype=BF16, device=gpu_device)
    starts = torch.tensor([69, 63], dtype=torch.int32, device=gpu_device)
    good = dict(query=q, cache=t.cache, starts=starts)
    hip_block_cache_attention(**good)
    for changes in (
        dict(query=q.half()), dict(query=q[:, :3]), dict(query=q[:1]), dict(query=q[..., :32]), dict(query=q.cpu()),
        dict(query=q[:, :0]), dict(query=torch.zeros(2, 4, 3, 68, dtype=BF16, device=gpu_device)[..., :64]),
        dict(starts=starts.long()), dict(starts=starts[:1]), dict(starts=None), dict(starts=starts.cpu()),
        dict(counts=starts.long()), dict(scale=math.inf), dict(max_length=-1), dict(query=q.clone().requires_grad_()),
    ):
        with pytest.raises(RuntimeError, match="ineligible"):
            hip_block_cache_attention(**{**good, **changes})
    kv = torch.zeros(2, 2, 1, 64, dtype=BF16, device=gpu_device)
    for key, value in ((kv[:, :1], kv[:, :1]), (kv, kv[:, :, :0]), (kv.half(), kv.half()), (kv, kv.float())):
        with pytest.raises(RuntimeError, match="ineligible"):
            hip_block_cache_append(t.cache, key, value, starts)
    for tokens in (-1, 2.0, True):
        with pytest.raises(RuntimeError, match="ineligible"):
            hip_block_cache_read(t.cache, starts, starts, tokens)


# ---------------------------------------------------------------------------
# the 4-bit linear layer


def _linear_case(device, rows, k, n, group, dtype, *, bias=True, gelu=False, seed=0):
    from solution.kernels.projection import hip_linear_w4, pack_linear_w4_codes

    generator = torch.Generator().manual_seed(seed)
    codes = torch.randint(-7, 8, (n, k), generator=generator)
    scales = (torch.rand(n, k // group, generator=generator) * 0.02 + 0.001).to(dtype)
    packed = pack_linear_w4_codes(codes.to(device), scales.to(device))
    x = _rand((rows, k), seed + 1, dtype)
    b = _rand((n,), seed + 2, dtype) if bias else None
    with torch.inference_mode():
        got, marker = hip_linear_w4(x.to(device), packed, None if b is None else b.to(device),
                                    activation="gelu" if gelu else "none")
    assert marker == "hip_linear_w4" and got.dtype == dtype
    weight = codes.double() * scales.double().repeat_interleave(group, dim=1)
    want, size = plain.linear(x.double(), weight, None if b is None else b.double(), gelu)
    _near(got, want, plain.linear_bound(want, size, k, gelu, dtype), f"linear {rows}x{k}x{n} group {group} {dtype}")


@pytest.mark.parametrize("rows", [1, 2, 13, 16, 17, 32, 33, 64, 65, 130])
@pytest.mark.parametrize("dtype,group", [(BF16, 32), (BF16, 128), (F16, 64)])
def test_linear_w4_rows(gpu_device, rows, dtype, group):
    _linear_case(gpu_device, rows, 640, 80, group, dtype, seed=rows)


@pytest.mark.parametrize("k,n", [(128, 16), (128, 4096), (1024, 48), (2176, 1024), (4096, 272), (16384, 32)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("gelu", [False, True])
def test_linear_w4_sizes(gpu_device, k, n, group, gelu):
    _linear_case(gpu_device, 3, k, n, group, BF16 if group != 64 else F16, bias=n != 48, gelu=gelu, seed=k + n)


@pytest.mark.parametrize("rows", [1, 9, 25, 50, 100])
@pytest.mark.parametrize("n", [16 * 512, 16 * 1024, 16 * 1026, 16 * 1027])
def test_linear_w4_wide(gpu_device, rows, n):
    """As many outputs as take two and four tiles of them a workgroup, or would."""

    _linear_case(gpu_device, rows, 384, n, 32 if rows == 50 else 128, F16 if rows == 9 else BF16, seed=rows)


def test_linear_w4_layouts_and_extremes(gpu_device):
    from solution.kernels.projection import hip_linear_w4, quantize_linear_w4

    weight = _rand((64, 256), 161, BF16).to(gpu_device)
    weight[3] = 0.0
    packed = quantize_linear_w4(weight, 32)
    wide = _rand((2, 3, 512), 162, BF16).to(gpu_device)
    with torch.inference_mode():
        x = wide[:, :, 128:384]
        assert torch.equal(hip_linear_w4(x, packed)[0], hip_linear_w4(x.contiguous(), packed)[0])
        one = wide[0, 0, :256]
        assert torch.equal(hip_linear_w4(one, packed)[0], hip_linear_w4(one[None], packed)[0][0])
        same = one.expand(5, 256)
        assert torch.equal(hip_linear_w4(same, packed)[0], hip_linear_w4(same.contiguous(), packed)[0])
        assert hip_linear_w4(wide[:0, :, :256], packed)[0].shape == (0, 3, 64)
        # a row's infinities and NaN stay in the row; large inputs lose nothing
        x = _rand((20, 256), 163, BF16).to(gpu_device)
        want = hip_linear_w4(x, packed)[0]
        x2 = x.clone()
        x2[4, 7], x2[18, 200] = math.nan, math.inf
        got = hip_linear_w4(x2, packed)[0]
        keep = [i for i in range(20) if i not in (4, 18)]
        assert torch.equal(got[keep], want[keep]) and bool(got[4].isnan().all())
        big = hip_linear_w4((x * 2.0**100).to(BF16), packed)[0]
        assert torch.equal(big, (want.float() * 2.0**100).to(BF16))
        with pytest.raises(RuntimeError, match="ineligible"):
            hip_linear_w4(wide.transpose(0, 1)[:, :, :256], packed)  # rows at two strides
    for x in (wide[..., :128], wide[..., :256].half(), wide[..., 4:260], wide[..., :256].cpu(),
              torch.zeros(2, 256, dtype=BF16, device=gpu_device).requires_grad_()):
        with pytest.raises(RuntimeError, match="ineligible"):
            hip_linear_w4(x, packed)
    for bias in (torch.zeros(32, dtype=BF16, device=gpu_device), torch.zeros(64, device=gpu_device)):
        with pytest.raises(RuntimeError, match="ineligible"):
            hip_linear_w4(one, packed, bias)
    with pytest.raises(RuntimeError, match="ineligible"):
        hip_linear_w4(one, packed, activation="relu")


@pytest.mark.parametrize("rows", [1, 5, 40])
@pytest.mark.parametrize("group", [32, 128])
def test_linear_w4_of_large_inputs(gpu_device, rows, group):
    """Inputs of up to bf16's largest: a group's sum of whole codes would leave fp32."""

    from solution.kernels.projection import hip_linear_w4, pack_linear_w4_codes

    generator = torch.Generator().manual_seed(rows)
    codes = torch.randint(-7, 8, (48, 256), generator=generator)
    codes[:16] = codes[:16].abs()  # sums without cancellation
    scales = torch.full((48, 256 // group), 2.0**-12).to(BF16)
    packed = pack_linear_w4_codes(codes.to(gpu_device), scales.to(gpu_device))
    x = (torch.rand((rows, 256), generator=generator) + 1).to(BF16) * 2.0**126
    with torch.inference_mode():
        got = hip_linear_w4(x.to(gpu_device), packed)[0]
    weight = codes.double() * 2.0**-12
    want, size = plain.linear(x.double(), weight, None, False)
    assert float(want.abs().max()) < torch.finfo(BF16).max
    _near(got, want, plain.linear_bound(want, size, 256, False, BF16), f"large inputs, {rows} rows")


# ---------------------------------------------------------------------------
# a decoding step


class _Layer:
    """One layer's attention branch with all four operators: 4-bit projections, the
    norm and rotation of heads, the cache and the attention over it."""

    def __init__(self, device, batch, heads, kv_heads, dim, dtype, max_tokens, seed=0):
        from solution.kernels.attention import BlockCache
        from solution.kernels.norm import rotary_table
        from solution.kernels.projection import quantize_linear_w4

        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        width = heads * dim
        self.width = width
        self.qkv = quantize_linear_w4(_rand(((heads + 2 * kv_heads) * dim, width), seed, dtype, width**-0.5).to(device), 64)
        self.out = quantize_linear_w4(_rand((width, width), seed + 1, dtype, width**-0.5).to(device), 64)
        self.bias = _rand(((heads + 2 * kv_heads) * dim,), seed + 2, dtype).to(device)
        self.wq, self.wk = (1 + _rand((dim,), seed + i, F32, 0.2).to(device) for i in (3, 4))
        self.table = rotary_table(max_tokens, dim, device=device)
        self.cache = BlockCache.allocate(batch, kv_heads, dim, max_tokens=max_tokens, dtype=dtype, device=device)

    def __call__(self, x, starts, counts=None):
        from solution.kernels.attention import hip_block_cache_append, hip_block_cache_attention
        from solution.kernels.norm import hip_qk_norm_rotary
        from solution.kernels.projection import hip_linear_w4

        batch, seq, _ = x.shape
        packed = hip_linear_w4(x, self.qkv, self.bias)[0].view(batch, seq, -1, self.dim)
        ends = self.heads, self.heads + self.kv_heads
        query, key, value = (t.transpose(1, 2) for t in packed.tensor_split(ends, dim=2))
        query, key, _ = hip_qk_norm_rotary(query, key, self.wq, self.wk, self.table, starts)
        hip_block_cache_append(self.cache, key, value, starts, counts)
        context, _ = hip_block_cache_attention(query, self.cache, starts, counts)
        return hip_linear_w4(context, self.out)[0], (packed, query, key, value, context)


def test_a_prompt_and_tokens_through_all_operators(gpu_device):
    """A ragged prompt, then token by token, every operator's answer against the
    plain form of what it was given."""

    batch, heads, kv_heads, dim = 3, 6, 2, 64
    layer = _Layer(gpu_device, batch, heads, kv_heads, dim, BF16, 400, seed=171)
    qkv, out_weight = (w.dequantize().double().cpu() for w in (layer.qkv, layer.out))
    starts = torch.zeros(batch, dtype=torch.int32, device=gpu_device)
    held = [[], [], []]  # (key, value) of each sequence so far
    for step, counts in enumerate([[130, 61, 1], None, None, None, [5, 1, 70], None]):
        seq = 1 if counts is None else max(counts)
        x = _rand((batch, seq, layer.width), 180 + step, BF16)
        counts_t = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=gpu_device)
        with torch.inference_mode():
            y, parts = layer(x.to(gpu_device), starts, counts_t)
        packed, query, key, value, context = (p.cpu() for p in parts)
        want, size = plain.linear(x.double().reshape(-1, layer.width), qkv, layer.bias.double().cpu(), False)
        _near(packed.reshape(want.shape), want, plain.linear_bound(want, size, layer.width, False, BF16), "projection")
        first = starts.cpu()
        for got, view, weight in ((query, packed[:, :, :heads], layer.wq), (key, packed[:, :, heads : heads + kv_heads], layer.wk)):
            want = plain.norm_rotary(view.transpose(1, 2).double(), weight.cpu(), None, layer.table.cpu(), first,
                                     norm="rms", eps=1e-6, interleaved=False)
            size = want.abs().amax(-1, keepdim=True) * 2 + 1
            _near(got, want, 2.0**-8 * want.abs() + 48 * 2.0**-24 * size, "norm and rotation")
        context = context.reshape(batch, seq, heads, dim)
        for b in range(batch):
            count = 1 if counts is None else counts[b]
            held[b].append((key[b, :, :count], value[b, :, :count]))
            all_key, all_value = (torch.cat([t[i] for t in held[b]], dim=1).double() for i in range(2))
            for h in (0, 2, 3, 5):
                keys, values = plain.stored_tokens(all_key[h // 3], all_value[h // 3])
                for i in {0, count // 2, count - 1}:
                    q, position = query[b, h, i].double(), int(first[b]) + i
                    want, size = plain.attention(q, keys, values, position, dim**-0.5)
                    bound = plain.attention_bound(want, size, q, keys, position, dim**-0.5, BF16)
                    _near(context[b, i, h], want, bound, f"step {step} sequence {b} head {h} row {i}")
        want, size = plain.linear(context.double().reshape(-1, layer.width), out_weight, None, False)
        _near(y.reshape(want.shape), want, plain.linear_bound(want, size, layer.width, False, BF16), "output projection")
        starts += torch.tensor(counts, dtype=torch.int32, device=gpu_device) if counts else 1


def test_captured_steps_replay_as_eager_ones(gpu_device):
    """Token after token from one captured graph, beside eager work: across the
    border of a block, against the same steps run eagerly."""

    batch = 4
    layers = [_Layer(gpu_device, batch, 8, 2, 64, BF16, 3000, seed=191) for _ in range(2)]
    prompt = _rand((batch, 123, 512), 192, BF16).to(gpu_device)
    tokens = [_rand((batch, 1, 512), 193 + i, BF16).to(gpu_device) for i in range(8)]
    with torch.inference_mode():
        zeros = torch.zeros(batch, dtype=torch.int32, device=gpu_device)
        for layer in layers:
            layer(prompt, zeros)
        starts = torch.full((batch,), 123, dtype=torch.int32, device=gpu_device)
        x = tokens[0].clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            y = layers[0](x, starts)[0]
            starts += 1
        torch.cuda.current_stream().wait_stream(stream)
        eager_starts = torch.full((batch,), 123, dtype=torch.int32, device=gpu_device)
        for i, token in enumerate(tokens):
            want = layers[1](token, eager_starts)[0]
            eager_starts += 1
            x.copy_(token)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want), f"step {i}"
        assert torch.equal(starts, eager_starts)
    for name in ("key_codes", "value_codes", "key_scales", "key_tail", "value_tail"):
        assert torch.equal(getattr(layers[0].cache, name), getattr(layers[1].cache, name)), name


def test_calls_without_tokens(gpu_device):
    """No sequences, no tokens, no rows: outputs of their shapes, and the cache as it was."""

    from solution.kernels.attention import BlockCache, hip_block_cache_append, hip_block_cache_attention, hip_block_cache_read
    from solution.kernels.norm import hip_qk_norm_rotary, rotary_table
    from solution.kernels.projection import hip_linear_w4, quantize_linear_w4

    weight = quantize_linear_w4(_rand((32, 128), 361, BF16).to(gpu_device))
    table = rotary_table(8, 64, device=gpu_device)
    with torch.inference_mode():
        for batch, seq in ((0, 3), (2, 0), (0, 0)):
            t = _Tokens(gpu_device, [70] * 2, 2, 64, BF16, seed=362).fill()
            cache = t.cache if batch else BlockCache.allocate(0, 2, 64, max_tokens=200, device=gpu_device)
            before = {n: getattr(t.cache, n).clone() for n in ("key_codes", "value_codes", "key_tail", "value_tail")}
            starts = torch.full((batch,), 70, dtype=torch.int32, device=gpu_device)
            q, kv = (torch.zeros(batch, h, seq, 64, dtype=BF16, device=gpu_device) for h in (4, 2))
            out = hip_qk_norm_rotary(q, kv, None, None, table, starts)
            assert out[0].shape == q.shape and out[1].shape == kv.shape
            hip_block_cache_append(cache, kv, kv, starts)
            assert hip_block_cache_attention(q, cache, starts)[0].shape == (batch, seq, 256)
            assert hip_block_cache_read(cache, starts, starts, seq)[0].shape == (batch, 2, seq, 64)
            assert hip_linear_w4(torch.zeros(batch, seq, 128, dtype=BF16, device=gpu_device), weight)[0].shape == (batch, seq, 32)
            for name, want in before.items():
                assert torch.equal(getattr(t.cache, name), want), name


@pytest.mark.parametrize("dim", [64, 128])
def test_captured_chunks_replay_as_eager_ones(gpu_device, dim):
    """Chunks in parts from one graph, at other places and of other lengths each time."""

    from solution.kernels.attention import hip_block_cache_append, hip_block_cache_attention

    seq, lengths = 90, [9_000, 4_000, 130]
    tokens = [_Tokens(gpu_device, lengths, 1, dim, BF16, seed=371) for _ in range(2)]
    for t in tokens:
        t.append([0] * 3, [8_000, 64, 0])
    query = _rand((3, 4, seq, dim), 372, BF16).to(gpu_device)
    kv = _rand((2, 3, 1, seq, dim), 373, BF16).to(gpu_device)
    to = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu_device)  # noqa: E731
    starts, counts = to([8_000, 64, 0]), to([seq, 1, 0])

    def step(cache, key, value, starts, counts):
        hip_block_cache_append(cache, key, value, starts, counts)
        return hip_block_cache_attention(query, cache, starts, counts)[0]

    with torch.inference_mode():
        key, value = kv[0].clone(), kv[1].clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            out = step(tokens[0].cache, key, value, starts, counts)
            starts += counts
        torch.cuda.current_stream().wait_stream(stream)
        held = [8_000, 64, 0]
        for i, new in enumerate(([seq, 1, 0], [3, 64, 20], [0, 0, 44], [64, seq, 1], [seq, 0, 65])):
            fresh = kv.roll(i, dims=3)
            want = step(tokens[1].cache, fresh[0], fresh[1], to(held), to(new))
            key.copy_(fresh[0]), value.copy_(fresh[1]), counts.copy_(to(new))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), i
            held = [a + b for a, b in zip(held, new)]
        assert starts.tolist() == held
    for name in ("key_codes", "value_codes", "key_scales", "value_scales", "key_tail", "value_tail"):
        assert torch.equal(getattr(tokens[0].cache, name), getattr(tokens[1].cache, name)), name


def test_two_streams_at_once(gpu_device):
    """Calls that overlap on two streams have workspaces of their own."""

    layers = [_Layer(gpu_device, 2, 8, 8, 64, BF16, 5000, seed=201 + i) for i in range(2)]
    x = _rand((2, 4000, 512), 203, BF16).to(gpu_device)
    token = _rand((2, 1, 512), 204, BF16).to(gpu_device)
    starts = torch.full((2,), 4000, dtype=torch.int32, device=gpu_device)
    with torch.inference_mode():
        for layer in layers:
            layer(x, torch.zeros_like(starts))
        want = [layer(token, starts)[0] for layer in layers]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in layers]
        got = [[], []]
        for _ in range(5):
            for layer, stream, out in zip(layers, streams, got):
                with torch.cuda.stream(stream):
                    out.append(layer(token, starts)[0])
        torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, y) for y in g)

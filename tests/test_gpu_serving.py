"""GPU parity of the operators around a decoding step with drafts against their plain
forms (tests/serving_reference.py), one by one and as a step runs them."""

from __future__ import annotations

import math

import pytest
import torch

import serving_reference as plain
from serving_reference import Book

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _generator(seed):
    return torch.Generator().manual_seed(seed)


def _rand(shape, seed, dtype, spread=1.0):
    return (torch.randn(shape, generator=_generator(seed)) * spread).to(dtype)


def _words(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


# ---------------------------------------------------------------------------
# verification


def _drafted(batch, drafts, vocab, dtype, seed, *, near=0.4, spread=2.0):
    """Target and draft logits that lie near each other, tokens drawn from the draft's
    probabilities, uniforms."""

    generator = _generator(seed)
    target = torch.randn((batch, drafts + 1, vocab), generator=generator) * spread
    draft = (target[:, :drafts] + near * torch.randn((batch, drafts, vocab), generator=generator)).to(dtype)
    noise = -torch.log(-torch.log(torch.rand(draft.shape, generator=generator).clamp(1e-30, 1 - 1e-7)))
    tokens = (draft.float() + noise).argmax(-1) if drafts else torch.zeros((batch, 0), dtype=torch.int64)
    uniforms = torch.rand((batch, drafts + 1), generator=generator)
    return target.to(dtype), draft, tokens, uniforms


def _verify(device, target, tokens, uniforms, draft=None, counts=None, temperatures=None, *, place=None):
    from solution.kernels.sampling import hip_verify_draft

    to = place or (lambda t: t.to(device))
    counts_t = None if counts is None else _words(counts, device)
    temperatures_t = None if temperatures is None else torch.tensor(temperatures, dtype=F32, device=device)
    with torch.inference_mode():
        answer, accepted, marker = hip_verify_draft(
            to(target), tokens.to(device), uniforms.to(device), None if draft is None else to(draft), counts=counts_t,
            temperatures=temperatures_t,
        )
    assert marker == "hip_verify_draft" and answer.dtype == torch.int64 and accepted.dtype == torch.int32
    want = plain.verify(
        target, tokens, uniforms, draft, counts,
        None if temperatures is None else torch.tensor(temperatures, dtype=F32),
    )
    assert accepted.tolist() == want[1]
    assert answer.tolist() == want[0]
    return want


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("vocab", [2, 63, 777, 8191, 8193, 50021])
def test_verify_types_and_vocabularies(gpu_device, dtype, sampled, vocab):
    target, draft, tokens, uniforms = _drafted(3, 4, vocab, dtype, vocab)
    _verify(gpu_device, target, tokens, uniforms, draft if sampled else None)


@pytest.mark.parametrize("batch,drafts", [(1, 0), (5, 0), (1, 1), (70, 2), (2, 16), (2, 40)])
@pytest.mark.parametrize("sampled", [True, False])
def test_verify_batches_and_drafts(gpu_device, batch, drafts, sampled):
    # near enough that long drafts stand in part
    target, draft, tokens, uniforms = _drafted(batch, drafts, 301, BF16, 7 + drafts, near=0.05)
    if not sampled:
        target = target * 4
        tokens = target[:, :drafts].float().argmax(-1)
    want = _verify(gpu_device, target, tokens, uniforms, draft if sampled else None)
    if drafts >= 16:
        assert max(want[1]) > 0


def test_verify_draws_from_the_target_alone_over_large_vocabularies(gpu_device):
    target, draft, tokens, uniforms = _drafted(2, 1, 200_003, BF16, 11, spread=0.2)
    _verify(gpu_device, target, tokens, uniforms, draft)
    _verify(gpu_device, target[:, :1], tokens[:, :0], uniforms[:, :1])


def test_verify_ragged_drafts_and_requests_without_part(gpu_device):
    target, draft, tokens, uniforms = _drafted(7, 3, 401, F16, 12)
    counts = [3, 0, 1, -1, 2, 9, -5]
    want = _verify(gpu_device, target, tokens, uniforms, draft, counts)
    assert want[1][3] == want[1][6] == -1 and want[0][3] == [-1] * 4
    _verify(gpu_device, target, tokens, uniforms, None, counts)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_verify_temperatures(gpu_device, dtype):
    temperatures = [0.0, 1.0, 0.3, 5.0, 1e-30, math.inf, -1.0, math.nan, 1e-45, 3e38]
    target, draft, tokens, uniforms = _drafted(len(temperatures), 3, 9001, dtype, 13, near=0.01)
    tokens[::2] = target[::2, :3].float().argmax(-1)
    target[3, :, 40:900] = -math.inf
    target[5, :, 17:4000] = -math.inf
    for given in (draft, None):
        _verify(gpu_device, target, tokens, uniforms, given, None, temperatures)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("size", [1e25, 1e31, 1e36])
def test_verify_large_logits_at_large_temperatures(gpu_device, dtype, sampled, size):
    target, draft, tokens, uniforms = _drafted(6, 3, 9001, F32, 22, near=0.1)
    target, draft = (target * size).to(dtype), (draft * size).to(dtype)
    target[2, :, 17:4000] = -math.inf
    temperatures = [size * t for t in (1.0, 0.5, 3.0, 1.0, 8.0, 1.5)]
    want = _verify(gpu_device, target, tokens, uniforms, draft if sampled else None, None, temperatures)
    assert len({row[0] for row in want[0]}) > 1


def test_verify_greedy_ties_take_the_lowest_token(gpu_device):
    target = torch.zeros((4, 3, 20_000), dtype=BF16)
    target[0, 0, [9000, 19_999]] = 3.0
    target[0, 1, [5, 8192]] = 2.0
    target[1, :, 12_345] = 1.0
    target[2, 0, [8191, 8192]] = 1.0
    tokens = torch.tensor([[9000, 8192], [12_345, 12_345], [8192, 0], [0, 0]])
    want = _verify(gpu_device, target, tokens, torch.full((4, 3), 0.5), None, None, [0.0] * 4)
    assert want == ([[9000, 5, -1], [12_345, 12_345, 12_345], [8191, -1, -1], [0, 0, 0]], [1, 2, 0, 2])


def test_verify_masked_logits_and_rows_without_a_distribution(gpu_device):
    target, draft, tokens, uniforms = _drafted(12, 2, 9000, F32, 14, near=0.0)
    inf, nan = math.inf, math.nan
    uniforms[:, 0] = 0.1
    target[0] = -inf
    target[0, :, 8500] = -3.0  # one token has it all
    draft[0], tokens[0] = target[0, :2], 8500
    target[1, 0] = -inf  # none
    target[2, 0, 777] = nan
    target[3, 0, 8999] = inf
    target[4, 1, 0] = nan  # met where the first draft stands
    draft[5, 0, 100] = nan
    draft[6, 0] = -inf
    draft[7, 0, 5] = inf
    target[8, 2, 5] = nan  # behind the first draft that does not stand
    uniforms[8] = 0.999999
    target[8, 0, tokens[8, 0]] = -40.0
    target[9, :, :8000] = -inf
    target[10, :, 8192:] = -inf
    target[11, 0, tokens[11, 0]] = draft[11, 0, tokens[11, 0]] = -inf  # no chance in either: nothing else to draw
    target[11, 0], draft[11, 0] = target[11, 0].clone(), target[11, 0].clone()
    want = _verify(gpu_device, target, tokens, uniforms, draft)
    assert want[0][0] == [8500, 8500, 8500]
    for b in (1, 2, 3, 5, 6, 7, 11):
        assert want[0][b][0] == -1 and want[1][b] == 0, b
    assert want[1][4] == 1 and want[0][4][1] == -1
    assert want[1][8] == 0 and want[0][8][0] >= 0
    _verify(gpu_device, target, tokens, uniforms)


def test_verify_drafts_outside_the_vocabulary(gpu_device):
    target, draft, tokens, uniforms = _drafted(5, 2, 50, BF16, 15)
    tokens[:, 0] = torch.tensor([-1, 50, 2**40, -(2**62), 49])
    uniforms[:, :2] = 0.0
    for given in (draft, None):
        want = _verify(gpu_device, target, tokens, uniforms, given)
        assert want[1][:4] == [0, 0, 0, 0]


@pytest.mark.parametrize("value", [0.0, 1e-38, 0.5, 1 - 2.0**-24, 1.0, 2.0, -1.0, math.nan])
def test_verify_extreme_random_numbers(gpu_device, value):
    """Numbers of [0, 1), and what others do: no draft stands on a NaN, and the draw ends
    at the last token with a weight."""

    target, draft, tokens, uniforms = _drafted(4, 2, 9000, BF16, 16)
    target[1, :, :100] = -math.inf
    target[2, :, 8000:] = -math.inf
    uniforms[:] = value
    _verify(gpu_device, target, tokens, uniforms, draft)
    _verify(gpu_device, target, tokens, uniforms)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("vocab", [50, 9001])
def test_verify_random_numbers_at_the_border(gpu_device, dtype, sampled, vocab):
    """Numbers next to p / q, where fp32 cannot say whether a draft stands: that of either
    side, in rows of which one after the other is so near."""

    batch, drafts = 24, 18
    target, draft, tokens, uniforms = _drafted(batch, drafts, vocab, dtype, 19 + vocab)
    if not sampled:
        tokens = target[:, :drafts].float().argmax(-1)
    p = torch.softmax(target[:, :drafts].double(), -1).gather(-1, tokens[..., None])[..., 0]
    q = torch.softmax(draft.double(), -1).gather(-1, tokens[..., None])[..., 0] if sampled else torch.ones_like(p)
    border = (p / q).clamp(max=0.999).float()
    step = torch.randint(-1, 2, border.shape, generator=_generator(20))
    step[:, : drafts // 2] = -1  # the first of them stand
    border = torch.where(step < 0, torch.nextafter(border, torch.zeros(())), border)
    uniforms[:, :drafts] = torch.where(step > 0, torch.nextafter(border, torch.ones(())), border)
    want = _verify(gpu_device, target, tokens, uniforms, draft if sampled else None)
    assert min(want[1]) >= drafts // 2 - 1 and min(want[1]) < drafts


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("batch,vocab", [(130, 50), (600, 50), (110, 9001)])
def test_verify_random_numbers_at_the_border_of_many_requests(gpu_device, dtype, sampled, batch, vocab):
    """As above, where the decision is the draw's launch's and where it has one of its own:
    numbers below p / q for the first drafts, on either side of it for the others."""

    drafts = 18
    target, draft, tokens, uniforms = _drafted(batch, drafts, vocab, dtype, 23 + vocab)
    if not sampled:
        tokens = target[:, :drafts].float().argmax(-1)
    p = torch.softmax(target[:, :drafts].double(), -1).gather(-1, tokens[..., None])[..., 0]
    q = torch.softmax(draft.double(), -1).gather(-1, tokens[..., None])[..., 0] if sampled else torch.ones_like(p)
    border = (p / q).clamp(max=0.999).float()
    step = torch.randint(-1, 2, border.shape, generator=_generator(24))
    step[:, : drafts // 2] = -1
    border = torch.where(step < 0, torch.nextafter(border, torch.zeros(())), border)
    uniforms[:, :drafts] = torch.where(step > 0, torch.nextafter(border, torch.ones(())), border)
    want = _verify(gpu_device, target, tokens, uniforms, draft if sampled else None)
    assert min(want[1]) >= drafts // 2 - 1 and min(want[1]) < drafts


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("batch", [128, 129, 512, 513, 1500])
def test_verify_of_many_requests_of_every_kind(gpu_device, batch, sampled):
    """Batches on both sides of where decision and draw become launches of their own."""

    generator = _generator(19)
    target, draft, tokens, uniforms = _drafted(batch, 3, 203, BF16, 20, near=0.1)
    if not sampled:
        tokens = target[:, :3].float().argmax(-1)
    counts = torch.randint(-1, 5, (batch,), generator=generator).tolist()
    temperatures = torch.tensor([1.0, 0.0, 0.4, math.inf, 1.0])[torch.randint(0, 5, (batch,), generator=generator)].tolist()
    target[::11, 1] = math.nan
    target[5::17, 0, 3:] = -math.inf
    draft[7::13, 0, 9] = math.inf
    tokens[9::19, 0] = 203
    want = _verify(gpu_device, target, tokens, uniforms, draft if sampled else None, counts, temperatures)
    assert set(want[1]) == {-1, 0, 1, 2, 3}


@pytest.mark.parametrize("batch,vocab", [(5, 777), (5, 50_021), (16, 131_073)])
@pytest.mark.parametrize("near", [1e-6, 1e-5, 1e-4, "one token"])
def test_verify_distributions_that_lie_close(gpu_device, batch, vocab, near):
    """p / q lies within 1e-6 .. 1e-4 of 1 for all tokens, or for all but a rare one, and
    max(p - q, 0) is as small: its tokens are those that the exact ratio of the two sums names."""

    generator = _generator(18)
    target = torch.randn((batch, 2, vocab), generator=generator) * 0.5
    if near == "one token":
        draft = target[:, :1].clone()
        tokens = torch.randint(0, vocab, (batch, 1), generator=generator)
        draft[torch.arange(batch), 0, tokens[:, 0]] += 1.0
    else:
        draft = target[:, :1] + near * torch.randn((batch, 1, vocab), generator=generator)
        tokens = (draft - target[:, :1]).argmax(-1)
    uniforms = torch.stack((torch.full((batch,), 1 - 2.0**-24), torch.rand((batch,), generator=generator)), dim=1)
    want = _verify(gpu_device, target, tokens, uniforms, draft)
    assert want[1] == [0] * batch and len({row[0] for row in want[0]}) > 1


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_verify_logits_of_any_strides(gpu_device, dtype):
    target, draft, tokens, uniforms = _drafted(3, 2, 1001, dtype, 17)
    want = _verify(gpu_device, target, tokens, uniforms, draft)

    def odd(t):  # columns of a wider tensor, rows beginning at any element
        wide = torch.full((*t.shape[:2], t.shape[2] + 6), math.nan, dtype=dtype, device=gpu_device)
        wide[..., 3:-3] = t.to(gpu_device)
        return wide[..., 3:-3]

    def turned(t):
        return t.transpose(0, 1).contiguous().to(gpu_device).transpose(0, 1)

    assert _verify(gpu_device, target, tokens, uniforms, draft, place=odd) == want
    assert _verify(gpu_device, target, tokens, uniforms, draft, place=turned) == want
    same = target[:, :1].expand(-1, 3, -1)
    _verify(gpu_device, same, tokens, uniforms, None, place=lambda t: t[:, :1].to(gpu_device).expand(-1, 3, -1))


def test_verify_of_more_than_four_gigabytes_of_logits(gpu_device):
    """Offsets beyond 32 bits: the answers of the last requests are those they have alone."""

    from solution.kernels.sampling import hip_verify_draft

    generator = torch.Generator(device=gpu_device).manual_seed(5)
    batch, drafts, vocab = 45, 3, 25_000_000
    row = torch.empty((2, drafts + 1, vocab), dtype=BF16, device=gpu_device).normal_(generator=generator)
    target = torch.zeros((batch, drafts + 1, vocab), dtype=BF16, device=gpu_device)
    target[-2:] = row
    tokens = torch.full((batch, drafts), vocab - 1, dtype=torch.int64, device=gpu_device)
    target[-1, :2, vocab - 1] = 40.0
    row[-1, :2, vocab - 1] = 40.0
    uniforms = torch.rand((batch, drafts + 1), device=gpu_device, generator=generator)
    with torch.inference_mode():
        got = hip_verify_draft(target, tokens, uniforms)
        want = hip_verify_draft(row, tokens[-2:], uniforms[-2:].contiguous())
    assert torch.equal(got[0][-2:], want[0]) and torch.equal(got[1][-2:], want[1])
    assert want[1].tolist()[-1] == 2


def test_verify_refusals(gpu_device):
    from solution.kernels.sampling import can_use_hip_verify_draft, hip_verify_draft

    target, draft, tokens, uniforms = (t.to(gpu_device) for t in _drafted(2, 3, 64, BF16, 18))
    assert can_use_hip_verify_draft(target, tokens, uniforms, draft)
    words = torch.zeros(2, dtype=torch.int32, device=gpu_device)
    heat = torch.ones(2, device=gpu_device)
    bad = (
        dict(target=target.double()),
        dict(target=target[0]),
        dict(target=target.transpose(1, 2)),
        dict(target=target[..., :0]),
        dict(target=target.clone().requires_grad_()),
        dict(tokens=tokens.int()),
        dict(tokens=tokens[:, :2]),
        dict(tokens=tokens.t().contiguous().t()),
        dict(tokens=None),
        dict(uniforms=uniforms.double()),
        dict(uniforms=uniforms[:, :3].contiguous()),
        dict(uniforms=uniforms.cpu()),
        dict(draft=draft.float()),
        dict(draft=draft[:, :2]),
        dict(draft=draft.transpose(0, 1)),
        dict(counts=words.long()),
        dict(counts=words[:1]),
        dict(temperatures=heat.double()),
        dict(temperatures=heat[:, None]),
    )
    for changes in bad:
        given = dict(target=target, tokens=tokens, uniforms=uniforms, draft=draft, counts=words, temperatures=heat)
        with pytest.raises(RuntimeError, match="ineligible"):
            hip_verify_draft(**{**given, **changes})
    empty = hip_verify_draft(target[:0], tokens[:0], uniforms[:0], draft[:0])
    assert empty[0].shape == (0, 4) and empty[1].shape == (0,)


# ---------------------------------------------------------------------------
# adapters


def _adapter_tensors(count, rank, k, n, dtype, seed, *, ranks=None, spread=1.0):
    down = _rand((count, rank, k), seed, dtype, spread * k**-0.5)
    up = _rand((count, n, rank), seed + 1, dtype, rank**-0.5)
    scales = torch.rand((count,), generator=_generator(seed + 2)) * 2 - 0.5
    if ranks is not None:  # zeros up to the next multiple of 8, anything behind
        for i, r in enumerate(ranks):
            last = -(-max(r, 0) // 8) * 8
            down[i, max(r, 0) : last], up[i, :, max(r, 0) : last] = 0, 0
            down[i, last:], up[i, :, last:] = math.nan, math.inf
    return down, up, scales


def _check_adapters(device, value, projected, down, up, scales, ranks, indices, counts=None, *, place=None, out=None):
    from solution.kernels.projection import LowRankAdapters, hip_low_rank_adapters

    to = place or (lambda t: t.to(device))
    packed = LowRankAdapters(
        down.to(device), up.to(device), None if scales is None else scales.to(device),
        None if ranks is None else _words(ranks, device),
    )
    given = to(projected)
    with torch.inference_mode():
        got, marker = hip_low_rank_adapters(
            to(value), given, packed, _words(indices, device), None if counts is None else _words(counts, device),
            out=given if out == "in place" else out,
        )
    assert marker == "hip_low_rank_adapters" and got.dtype == value.dtype and got.shape == projected.shape
    if out == "in place":
        assert got is given
    three = (lambda t: t[:, None] if t.ndim == 2 else t)  # noqa: E731
    want, terms, hidden = plain.adapters(three(value), three(projected), down, up, scales,
                                         None if ranks is None else torch.tensor(ranks), torch.tensor(indices), counts)
    bound = plain.adapters_bound(want, terms, hidden, value.shape[-1], down.shape[1], value.dtype)
    got = three(got).double().cpu()
    exact = (terms == 0) & (hidden == 0)
    assert torch.equal(got[exact], want[exact]), "rows without an adapter changed"
    assert torch.isfinite(got).all()
    off = (got - want).abs() - bound
    assert float(off.max()) <= 0 if off.numel() else True, float(off.max())
    return got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 128])
@pytest.mark.parametrize("seq", [1, 21])
def test_adapters_types_and_ranks(gpu_device, dtype, rank, seq):
    down, up, scales = _adapter_tensors(3, rank, 136, 200, dtype, rank)
    value, projected = _rand((4, seq, 136), 31, dtype), _rand((4, seq, 200), 32, dtype)
    _check_adapters(gpu_device, value, projected, down, up, scales, None, [2, 0, -1, 2])


@pytest.mark.parametrize("k,n", [(8, 8), (24, 1032), (32, 64), (520, 8), (1000, 1160), (4096, 72), (8200, 40)])
@pytest.mark.parametrize("batch,seq", [(1, 1), (3, 17), (2, 8200)])
def test_adapters_sizes(gpu_device, k, n, batch, seq):
    """Few tokens, whose products two launches share, and many, of which a wave does both."""

    if seq > 1000 and k * n > 100_000:
        k, n = min(k, 520), min(n, 136)
    down, up, scales = _adapter_tensors(2, 16, k, n, BF16, k + n)
    value, projected = _rand((batch, seq, k), 33, BF16), _rand((batch, seq, n), 34, BF16)
    _check_adapters(gpu_device, value, projected, down, up, scales, None, [i % 2 for i in range(batch)])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("seq", [1, 40, 4000])
def test_adapters_of_mixed_ranks_and_ragged_rows(gpu_device, dtype, seq):
    """Ranks that end inside a tile or leave nothing; NaN and infinities in what lies behind them."""

    ranks = [64, 1, 17, 0, 33, -3, 200, 48]
    down, up, scales = _adapter_tensors(8, 64, 104, 136, dtype, 35, ranks=ranks)
    indices = [0, 1, 2, 3, 4, 5, 6, 7, -1, 8, 2**31 - 1, 2, 2]
    counts = [seq, seq + 5, seq, seq, 1, seq, seq - 1, seq, seq, seq, seq, 0, -4]
    value, projected = _rand((13, seq, 104), 36, dtype), _rand((13, seq, 136), 37, dtype)
    _check_adapters(gpu_device, value, projected, down, up, scales, ranks, indices, counts)
    _check_adapters(gpu_device, value, projected, down, up, None, ranks, indices, counts, out="in place")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rank", [8, 32, 40, 64, 128])
@pytest.mark.parametrize("seq,k,n", [(1, 2056, 200), (21, 4104, 72), (70, 520, 8200), (3, 16384, 16)])
def test_adapters_of_few_tokens_and_long_rows(gpu_device, dtype, rank, seq, k, n):
    """Inputs or outputs that two launches share, mixed ranks, ragged rows, strides, in place."""

    ranks = [rank, rank - 7, 0, 200]
    down, up, scales = _adapter_tensors(4, rank, k, n, dtype, 57, ranks=ranks)
    indices, counts = [0, 1, 2, 3, -1, 1, 0], [seq, seq + 1, seq, seq - 1, seq, 0, 2]
    value, projected = _rand((7, seq, k), 58, dtype), _rand((7, seq, n), 59, dtype)
    _check_adapters(gpu_device, value, projected, down, up, scales, ranks, indices, counts)
    turned = (lambda t: t.transpose(0, 1).contiguous().to(gpu_device).transpose(0, 1))  # noqa: E731
    _check_adapters(gpu_device, value, projected, down, up, None, ranks, indices, counts, place=turned, out="in place")


@pytest.mark.parametrize("dtype,rank", [(BF16, 16), (F16, 72)])
def test_adapters_of_outputs_larger_than_the_caches(gpu_device, dtype, rank):
    ranks = [rank, rank - 9, 0]
    down, up, scales = _adapter_tensors(3, rank, 40, 4096, dtype, 60, ranks=ranks)
    value, projected = _rand((4, 4500, 40), 61, dtype), _rand((4, 4500, 4096), 62, dtype)
    for out in (None, "in place"):
        _check_adapters(gpu_device, value, projected, down, up, scales, ranks, [1, 2, 0, -1], [4500, 4500, 33, 7], out=out)


@pytest.mark.parametrize("batch", [1023, 1024, 1100])
def test_adapters_of_one_token_of_many_requests(gpu_device, batch):
    down, up, scales = _adapter_tensors(50, 16, 64, 72, F16, 38)
    indices = torch.randint(-1, 50, (batch,), generator=_generator(39)).tolist()
    value, projected = _rand((batch, 64), 40, F16), _rand((batch, 72), 41, F16)
    _check_adapters(gpu_device, value, projected, down, up, scales, None, indices)


@pytest.mark.parametrize("seq", [5, 9000])
def test_adapters_on_views_and_in_place(gpu_device, seq):
    """Rows of a packed projection, tokens outermost, one row for all; outputs into part of
    another tensor, whose rest stays."""

    down, up, scales = _adapter_tensors(2, 16, 64, 72, BF16, 42)
    value, projected = _rand((2, seq, 64), 43, BF16), _rand((2, seq, 72), 44, BF16)

    def packed(t):
        wide = torch.full((2, seq, t.shape[2] + 24), math.nan, dtype=BF16, device=gpu_device)
        wide[..., 8:-16] = t.to(gpu_device)
        return wide[..., 8:-16]

    def turned(t):
        return t.transpose(0, 1).contiguous().to(gpu_device).transpose(0, 1)

    want = _check_adapters(gpu_device, value, projected, down, up, scales, None, [1, 0])
    for place in (packed, turned):
        for out in (None, "in place"):
            got = _check_adapters(gpu_device, value, projected, down, up, scales, None, [1, 0], place=place, out=out)
            assert torch.equal(got, want)
    wide = torch.full((2, seq, 104), 7.0, dtype=BF16, device=gpu_device)
    got = _check_adapters(gpu_device, value, projected, down, up, scales, None, [1, 0], [seq, 2], out=wide[..., 16:88])
    assert torch.equal(wide[..., 16:88].double().cpu(), got)
    assert wide[..., :16].eq(7).all() and wide[..., 88:].eq(7).all()
    same = value[:, :1].expand(-1, seq, -1)
    _check_adapters(gpu_device, same, projected, down, up, scales, None, [1, 0],
                    place=lambda t: t[:, :1].to(gpu_device).expand(-1, seq, -1) if t is same else t.to(gpu_device))


@pytest.mark.parametrize("seq", [3, 9000])
@pytest.mark.parametrize("dtype,size", [(F16, 1e3), (F16, 1e-4), (BF16, 1e15), (BF16, 1e-15)])
def test_adapters_of_large_and_small_products(gpu_device, seq, dtype, size):
    """x down beyond fp16's range, or below it, with up and scale that bring it back."""

    value, projected = _rand((2, seq, 64), 45, dtype, size), _rand((2, seq, 72), 46, dtype)
    down, up, _ = _adapter_tensors(2, 24, 64, 72, dtype, 47, spread=1e3 if size > 1 else 1e-2)
    scales = torch.tensor([1.0, -0.5]) / (size * (1e3 if size > 1 else 1e-2))
    _check_adapters(gpu_device, value, projected, down, up, scales, None, [0, 1])


@pytest.mark.parametrize("dtype,bits", [(BF16, 24), (F16, 22)])
@pytest.mark.parametrize("rank", [16, 64, 128])
@pytest.mark.parametrize("seq,k,n", [(1, 24, 72), (20, 4104, 136), (9000, 24, 72), (17_000, 24, 4096)])
def test_adapters_whose_middle_factors_differ_in_the_last_bits(gpu_device, dtype, bits, rank, seq, k, n):
    """Directions in pairs with h = a + b + c and a + b, of which an output takes the
    difference c: whole numbers (times 2^-12) of up to ``bits`` bits whose every sum fp32
    holds, so the answer is exact where h reaches the second product with all its bits."""

    from solution.kernels.projection import LowRankAdapters, hip_low_rank_adapters

    last = bits - 16
    down, up = torch.zeros((1, rank, k)), torch.zeros((1, n, rank))
    pairs = rank // 2
    draw = lambda low, high: torch.randint(low, high, (pairs,), generator=_generator(48 + rank)).float()  # noqa: E731
    first, middle, least = draw(128, 256) * 2.0 ** (8 + last), draw(128, 256) * 2.0**last, draw(2 ** (last - 1), 2**last)
    for place, part in ((0, first), (k // 2, middle), (k - 1, least)):
        down[0, 0::2, place] = down[0, 1::2, place] = part * 2.0**-12
    down[0, 1::2, k - 1] = 0
    taken = torch.arange(n) % pairs
    up[0, torch.arange(n), 2 * taken], up[0, torch.arange(n), 2 * taken + 1] = 1.0, -1.0
    given = [t.to(dtype) for t in (torch.ones(1, seq, k), torch.zeros(1, seq, n), down, up)]
    assert torch.equal(given[2].float(), down)
    value, projected, down, up = (t.to(gpu_device) for t in given)
    with torch.inference_mode():
        got = hip_low_rank_adapters(value, projected, LowRankAdapters(down, up), _words([0], gpu_device))[0]
    want = (least[taken] * 2.0**-12).to(dtype).to(gpu_device)
    assert torch.equal(got, want.expand(1, seq, n))


@pytest.mark.parametrize("seq,features", [(20, 64), (9000, 64), (20, 4096)])
def test_adapters_keep_bad_tokens_to_themselves(gpu_device, seq, features):
    from solution.kernels.projection import LowRankAdapters, hip_low_rank_adapters

    down, up, scales = (t.to(gpu_device) for t in _adapter_tensors(2, 16, features, 72, BF16, 48))
    value, projected = _rand((2, seq, features), 49, BF16).to(gpu_device), _rand((2, seq, 72), 50, BF16).to(gpu_device)
    packed, indices = LowRankAdapters(down, up, scales), _words([0, 1], gpu_device)
    with torch.inference_mode():
        want = hip_low_rank_adapters(value, projected, packed, indices)[0]
        value[0, 7, 3], value[1, 2, 0] = math.nan, math.inf
        value[1, 18:] = math.nan  # behind the sequence's tokens
        got = hip_low_rank_adapters(value, projected, packed, indices, _words([seq, 18], gpu_device))[0]
    assert got[0, 7].isnan().all() and not got[1, 2].isfinite().any()
    want = want.clone()
    want[0, 7], want[1, 2], want[1, 18:] = got[0, 7], got[1, 2], projected[1, 18:]
    assert torch.equal(got.nan_to_num(9.0), want.nan_to_num(9.0))


def _run_adapters(device, value, projected, down, up, ranks=None):
    """One adapter's outputs on the CPU."""

    from solution.kernels.projection import LowRankAdapters, hip_low_rank_adapters

    packed = LowRankAdapters(down.to(device), up.to(device), None, None if ranks is None else _words(ranks, device))
    indices = _words([0] * value.shape[0], device)
    with torch.inference_mode():
        return hip_low_rank_adapters(value.to(device), projected.to(device), packed, indices)[0].cpu()


def _same_with_infinities(got, want):
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(0.5, 1e30, -1e30), want.nan_to_num(0.5, 1e30, -1e30))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("seq,k,n", [(1, 24, 72), (20, 4104, 136), (9000, 24, 72), (17_000, 24, 4096)])
def test_adapters_with_an_infinite_middle_factor(gpu_device, dtype, seq, k, n):
    """A weight of `down` is infinite, and with it one direction's h, beside others of 2^24,
    beyond fp16's range: infinite outputs of its sign, NaN where its input is 0."""

    down, up, value = torch.zeros((1, 16, k)), torch.zeros((1, n, 16)), torch.zeros((1, seq, k))
    down[0, 0, 0], down[0, 1:, k - 1] = math.inf, 512.0
    up[0, :, 0] = torch.where(torch.arange(n) % 3 == 0, -0.25, 2.0)
    up[0, :, 1] = torch.where(torch.arange(n) % 2 == 0, -1.0, 1.0)
    value[0, :, 0] = torch.tensor([1.0, -1.0, 0.5, 0.0])[torch.arange(seq) % 4]
    value[0, :, k - 1] = 2.0**15
    projected = _rand((1, seq, n), 96, dtype)
    got = _run_adapters(gpu_device, value.to(dtype), projected, down.to(dtype), up.to(dtype))
    want = (value[0, :, :1] * math.inf) * up[0, :, 0]
    assert float(want[0, 0]) == -math.inf and float(want[0, 1]) == math.inf
    _same_with_infinities(got[0].float(), want)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rank,own", [(16, None), (16, 7), (64, 24), (128, None), (128, 100)])
@pytest.mark.parametrize("seq,k,n", [(1, 24, 72), (3, 24, 72), (20, 4104, 136), (9000, 24, 72), (17_000, 24, 4096)])
def test_adapters_with_infinite_weights_of_the_outputs(gpu_device, dtype, rank, own, seq, k, n):
    """Weights of `up` are infinite: outputs of the sign of their direction's h, NaN where two
    of different signs meet and for an h of 0, and all others as they are without these."""

    own = own or rank
    down, up = torch.zeros((1, rank, k)), _rand((1, n, rank), 97, F32, own**-0.5)
    down[0, :own] = _rand((own, k), 98, F32, k**-0.5)
    up[0, :, own : -(-own // 8) * 8] = 0
    value, projected = _rand((1, seq, k), 99, dtype), _rand((1, seq, n), 100, dtype)
    value[0, 3 * seq // 4] = 0  # an h of 0
    down, up = down.to(dtype), up.to(dtype)
    ranks = None if own == rank else [own]
    want = _run_adapters(gpu_device, value, projected, down, up, ranks)
    bad = up.clone()
    bad[0, 1, 0], bad[0, 5, own - 1], bad[0, 8, [0, 2]] = math.inf, -math.inf, math.inf
    h = value[0].double() @ down[0].double().t()
    sign = h[:, [0, 2, own - 1]].sign()
    # (an h so near 0 that fp32's sums may miss its sign stays out)
    sure = (h[:, [0, 2, own - 1]].abs() > (k + 8) * 2.0**-24 * (value[0].double().abs() @ down[0].double().abs().t())[:, [0, 2, own - 1]]).all(1)
    sure[3 * seq // 4] = True
    assert sure.sum() > 0.5 * seq
    want = want[0].float()
    want[:, 1], want[:, 5] = (sign[:, 0] * math.inf).float(), (-sign[:, 2] * math.inf).float()
    want[:, 8] = (sign[:, 0] * math.inf + sign[:, 1] * math.inf).float()
    got = _run_adapters(gpu_device, value, projected, down, bad, ranks)[0].float()
    _same_with_infinities(got[sure], want[sure])


def test_adapters_of_more_than_four_gigabytes(gpu_device):
    """Offsets beyond 32 bits in the weights, the inputs and the outputs."""

    from solution.kernels.projection import LowRankAdapters, hip_low_rank_adapters

    count, rank, k, n = 300, 128, 65_536, 8192  # down of 5 GB
    down = torch.zeros((count, rank, k), dtype=BF16, device=gpu_device)
    up = torch.zeros((count, n, rank), dtype=BF16, device=gpu_device)
    small = [t.to(gpu_device) for t in _adapter_tensors(1, rank, k, n, BF16, 51)[:2]]
    down[-1], up[-1] = small[0][0], small[1][0]
    value, projected = _rand((2, 3, k), 52, BF16).to(gpu_device), _rand((2, 3, n), 53, BF16).to(gpu_device)
    with torch.inference_mode():
        got = hip_low_rank_adapters(value, projected, LowRankAdapters(down, up), _words([299, 0], gpu_device))[0]
        want = hip_low_rank_adapters(value, projected, LowRankAdapters(*small), _words([0, -1], gpu_device))[0]
    assert torch.equal(got, want) and not torch.equal(got[0], projected[0])
    del down, up, small
    long = 300_000  # tokens: x and y of 5 GB
    down, up, scales = (t.to(gpu_device) for t in _adapter_tensors(1, 8, 8192, 8192, BF16, 54))
    value = torch.zeros((1, long, 8192), dtype=BF16, device=gpu_device)
    projected = torch.zeros((1, long, 8192), dtype=BF16, device=gpu_device)
    value[0, -40:], projected[0, -40:] = _rand((40, 8192), 55, BF16).to(gpu_device), _rand((40, 8192), 56, BF16).to(gpu_device)
    with torch.inference_mode():
        packed, first = LowRankAdapters(down, up, scales), _words([0], gpu_device)
        got = hip_low_rank_adapters(value, projected, packed, first)[0][0, -40:].clone()
    _check_adapters(gpu_device, value[:, -40:].cpu(), projected[:, -40:].cpu(), down.cpu(), up.cpu(), scales.cpu(), None, [0])
    want, terms, hidden = plain.adapters(value[:, -40:].cpu(), projected[:, -40:].cpu(), down.cpu(), up.cpu(), scales.cpu(),
                                         None, torch.tensor([0]), None)
    bound = plain.adapters_bound(want, terms, hidden, 8192, 8, BF16)
    assert ((got.double().cpu() - want[0]).abs() <= bound[0]).all()


def test_adapters_refusals(gpu_device):
    from solution.kernels.projection import LowRankAdapters, can_use_hip_low_rank_adapters, hip_low_rank_adapters

    down, up, scales = (t.to(gpu_device) for t in _adapter_tensors(2, 16, 64, 72, BF16, 57))
    packed = LowRankAdapters(down, up, scales)
    value, projected = _rand((2, 3, 64), 58, BF16).to(gpu_device), _rand((2, 3, 72), 59, BF16).to(gpu_device)
    indices = _words([0, 1], gpu_device)
    assert can_use_hip_low_rank_adapters(value, projected, packed, indices)
    bad = (
        dict(value=value.half()),
        dict(value=value[..., :56]),
        dict(value=value.cpu()),
        dict(value=value[None]),
        dict(value=value.transpose(1, 2).contiguous().transpose(1, 2)),
        dict(value=value.clone().requires_grad_()),
        dict(projected=projected[..., :64]),
        dict(projected=projected.float()),
        dict(projected=projected[:, :2]),
        dict(indices=indices.long()),
        dict(indices=indices[:1]),
        dict(indices=None),
        dict(counts=indices.long()),
    )
    for changes in bad:
        given = dict(value=value, projected=projected, adapters=packed, indices=indices, counts=indices)
        with pytest.raises(RuntimeError, match="ineligible"):
            hip_low_rank_adapters(**{**given, **changes})
    wide = torch.zeros((2, 3, 144), dtype=BF16, device=gpu_device)
    square = torch.zeros((2, 3, 64), dtype=BF16, device=gpu_device)
    square_adapters = LowRankAdapters(down, up[:, :64].contiguous(), scales)
    outs = (
        (value, projected, packed, wide[..., :64]),
        (value, projected, packed, wide[..., :72].float()),
        (value, projected, packed, wide[..., 4:76]),
        (value, projected, packed, projected[:, :1].expand(-1, 3, -1)),
        (value, wide[..., :72], packed, wide[..., 72:]),  # rows between the input's
        (square, square.clone(), square_adapters, square),  # over the projection's input
    )
    for x, y, adapters, out in outs:
        with pytest.raises(RuntimeError, match="output buffer"):
            hip_low_rank_adapters(x, y, adapters, indices, out=out)
    with pytest.raises(RuntimeError, match="execution failed"):  # rows of the output that overlap
        hip_low_rank_adapters(value, projected, packed, indices, out=wide[0, :1, :72].expand(2, 3, -1))
    with torch.inference_mode():
        for shape in ((0, 3), (2, 0)):
            x, y = value[: shape[0], : shape[1]], projected[: shape[0], : shape[1]]
            assert hip_low_rank_adapters(x, y, packed, indices[: shape[0]])[0].shape == y.shape
        none = LowRankAdapters(down[:0], up[:0], scales[:0])
        assert torch.equal(hip_low_rank_adapters(value, projected, none, indices)[0], projected)


# ---------------------------------------------------------------------------
# the pool


def _pool(device, table, holders=None, num_blocks=None):
    from solution.kernels.attention import BlockPool

    table = _words(table, device).reshape(len(table), -1) if table else _words([], device).reshape(0, 4)
    if holders is None:
        return BlockPool.from_table(table, num_blocks)
    return BlockPool(table, _words(holders, device))


def _same_book(pool, book, what=""):
    assert pool.block_table.tolist() == book.table, what
    assert pool.holders.tolist() == book.holders, what


def _random_pool(device, batch, width, blocks, seed):
    """A table of some blocks of every sequence, some of them shared, and the lengths."""

    generator = _generator(seed)
    order = torch.randperm(blocks, generator=generator).tolist()
    lengths = torch.randint(0, width * 64 + 64, (batch,), generator=generator).tolist()
    table = [[-1] * width for _ in range(batch)]
    for b in range(batch):
        for j in range(min(lengths[b] // 64, width)):
            if b and j < lengths[b - 1] // 64 and j < 2 and int(torch.randint(0, 2, (1,), generator=generator)):
                table[b][j] = table[b - 1][j]
            elif order:
                table[b][j] = order.pop()
    pool = _pool(device, table, num_blocks=blocks)
    return pool, Book(pool.block_table.tolist(), pool.holders.tolist()), lengths


@pytest.mark.parametrize("batch,width,blocks,tokens", [
    (1, 1, 1, 1), (3, 5, 40, 1), (70, 3, 300, 64), (9, 40, 200, 700), (5, 130, 700, 9000), (2, 4, 0, 64), (3, 0, 5, 200),
    (1500, 2, 2500, 65),
])
def test_reserve(gpu_device, batch, width, blocks, tokens):
    from solution.kernels.attention import hip_block_pool_reserve

    pool, book, lengths = _random_pool(gpu_device, batch, width, blocks, batch + blocks)
    counts = torch.randint(-1, tokens + 9, (batch,), generator=_generator(61)).tolist()
    if batch > 4:
        lengths[3] = -5
    for given in (counts, None):
        missing, marker = hip_block_pool_reserve(
            pool, _words(lengths, gpu_device), tokens, None if given is None else _words(given, gpu_device)
        )
        assert marker == "hip_block_pool_reserve"
        assert missing.tolist() == book.reserve(lengths, tokens, given)
        _same_book(pool, book)


def test_reserve_takes_the_lowest_of_many_places(gpu_device):
    """Free places behind whole passes of held ones, and beyond 2^16."""

    from solution.kernels.attention import hip_block_pool_reserve

    holders = torch.ones(100_003, dtype=torch.int32)
    holders[[16_383, 16_384, 70_000, 99_999, 100_002]] = 0
    for tokens, want in ((63, 0), (64, 1), (6 * 64 + 1, 6)):
        pool = _pool(gpu_device, [[-1] * 7, [5] * 7], holders.tolist())
        missing, _ = hip_block_pool_reserve(pool, _words([0, 0], gpu_device), tokens)
        free = [16_383, 16_384, 70_000, 99_999, 100_002]
        assert pool.block_table[0].tolist() == (free + [-1] * 7)[:want] + [-1] * (7 - want) if want <= 5 else True
        assert missing.tolist() == [max(0, want - 5), 0]
        assert int(pool.holders.sum()) == 99_998 + min(want, 5)


@pytest.mark.parametrize("blocks", [5, 6, 7])
def test_reserve_that_runs_out_part_way(gpu_device, blocks):
    from solution.kernels.attention import hip_block_pool_reserve

    free = [16_383, 16_384, 70_000, 99_999, 100_002]
    holders = torch.ones(100_003, dtype=torch.int32)
    holders[free] = 0
    pool = _pool(gpu_device, [[-1] * 7, [-1] * 7, [5] * 7], holders.tolist())
    missing, _ = hip_block_pool_reserve(pool, _words([0, 0, 0], gpu_device), blocks * 64, _words([blocks * 64, 64, 9], gpu_device))
    assert pool.block_table.tolist() == [free + [-1] * 2, [-1] * 7, [5] * 7]
    assert missing.tolist() == [blocks - 5, 1, 0]
    holders[free] = 1
    assert torch.equal(pool.holders.cpu(), holders)


def test_reserve_of_far_positions(gpu_device):
    from solution.kernels.attention import hip_block_pool_reserve

    pool = _pool(gpu_device, [[-1] * 3] * 3, [0] * 4)
    starts = [2**31 - 2, 128, 190]
    missing, _ = hip_block_pool_reserve(pool, _words(starts, gpu_device), 2**31 - 1)
    last = [(s + 2**31 - 1) // 64 for s in starts]
    assert missing.tolist() == [last[0] - starts[0] // 64, last[1] - 3, last[2] - 3]
    assert pool.block_table.tolist() == [[-1] * 3, [-1, -1, 0], [-1, -1, 1]]
    missing, _ = hip_block_pool_reserve(pool, _words(starts, gpu_device), 0)
    assert missing.tolist() == [0, 0, 0]


@pytest.mark.parametrize("batch,width,blocks", [(1, 1, 3), (6, 9, 60), (300, 5, 900), (3, 600, 2000)])
def test_release(gpu_device, batch, width, blocks):
    from solution.kernels.attention import hip_block_pool_release

    pool, book, lengths = _random_pool(gpu_device, batch, width, blocks, 62 + batch)
    keep = [max(-1, n - int(d)) for n, d in zip(lengths, torch.randint(-100, 300, (batch,), generator=_generator(63)))]
    assert hip_block_pool_release(pool, _words(keep, gpu_device)) == "hip_block_pool_release"
    book.release(keep)
    _same_book(pool, book)
    hip_block_pool_release(pool, _words([0] * batch, gpu_device))
    assert pool.block_table.eq(-1).all() and pool.holders.eq(0).all()


@pytest.mark.parametrize("batch,width,blocks", [(1, 2, 3), (4, 11, 60), (64, 40, 3000), (1024, 3, 4000), (257, 17, 5000)])
def test_fork_of_the_table(gpu_device, batch, width, blocks):
    """Sequences that change places, are copied several times, or named from outside."""

    from solution.kernels.attention import hip_block_pool_fork

    pool, book, lengths = _random_pool(gpu_device, batch, width, blocks, 64 + batch)
    for seed in range(3):
        sources = torch.randint(0, batch, (batch,), generator=_generator(seed)).tolist()
        sources[0] = -1 if seed == 1 else batch if seed == 2 else batch - 1
        if batch > 3:
            sources[1], sources[2] = 2, 1
        assert hip_block_pool_fork(pool, _words(sources, gpu_device), _words(lengths, gpu_device)) == "hip_block_pool_fork"
        book.fork(sources, lengths)
        _same_book(pool, book, seed)
        lengths = [lengths[s] if 0 <= s < batch else n for s, n in zip(sources, lengths)]
    hip_block_pool_fork(pool, _words([batch - 1] * batch, gpu_device), _words([-7] * batch, gpu_device))
    book.fork([batch - 1] * batch, [-7] * batch)
    _same_book(pool, book)


@pytest.mark.parametrize("batch,width,blocks", [(1, 1, 1), (2, 3, 7), (6, 9, 60), (70, 30, 2500), (20, 900, 40_000), (3, 4, 0), (0, 4, 5)])
def test_compact(gpu_device, batch, width, blocks):
    from solution.kernels.attention import hip_block_pool_compact, hip_block_pool_release

    pool, book, lengths = _random_pool(gpu_device, batch, width, blocks, 65 + batch)
    ended = [0 if b % 3 == 1 else -1 for b in range(batch)]
    hip_block_pool_release(pool, _words(ended, gpu_device))
    book.release(ended)
    for again in range(2):
        origins, used, marker = hip_block_pool_compact(pool)
        want = book.compact()
        assert marker == "hip_block_pool_compact"
        assert (origins.tolist(), used.tolist()) == (want[0], [want[1]])
        _same_book(pool, book, again)
    assert not any(p >= 0 for p in want[0])  # nothing is left to move


def test_pool_with_entries_outside_it(gpu_device):
    """Places that are none hold nothing and are given up, reserved and kept as such."""

    from solution.kernels.attention import (
        hip_block_pool_compact, hip_block_pool_fork, hip_block_pool_release, hip_block_pool_reserve,
    )

    table = [[9, -7, 0, 2**31 - 1], [3, 4, -2, 5], [1, 1, 1, 1]]
    holders = [1, 4, 0, 1, 0]
    calls = (
        (hip_block_pool_reserve, ([64, 64, 0], 100), lambda book: book.reserve([64, 64, 0], 100)),
        (hip_block_pool_release, ([64, 128, -1],), lambda book: book.release([64, 128, -1])),
        (hip_block_pool_fork, ([1, 0, 0], [256, 100, 0]), lambda book: book.fork([1, 0, 0], [256, 100, 0])),
        (hip_block_pool_compact, (), lambda book: book.compact()),
    )
    for call, args, of_book in calls:
        pool, book = _pool(gpu_device, table, holders), Book(table, holders)
        call(pool, *(_words(a, gpu_device) if isinstance(a, list) else a for a in args))
        of_book(book)
        _same_book(pool, book, call.__name__)


# ---------------------------------------------------------------------------
# data of the cache


_CODES = ("key_codes", "value_codes", "key_scales", "value_scales")


def _filled_cache(device, batch, heads, dim, dtype, blocks, table, seed):
    """A cache whose places hold any codes and whose tails any values."""

    from solution.kernels.attention import BlockCache

    table = _words(table, device).reshape(batch, -1)
    cache = BlockCache.allocate(batch, heads, dim, max_tokens=0, num_blocks=blocks, dtype=dtype, device=device, block_table=table)
    generator = torch.Generator(device=device).manual_seed(seed)
    for codes in (cache.key_codes, cache.value_codes):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=generator, device=device))
    for scales in (cache.key_scales, cache.value_scales):
        scales.copy_(2.0 ** torch.randint(-9, 3, scales.shape, generator=generator, device=device))
    for tail in (cache.key_tail, cache.value_tail):
        tail.copy_(torch.randn(tail.shape, generator=generator, device=device))
    return cache


@pytest.mark.parametrize("heads,dim,blocks", [(1, 64, 9), (3, 128, 40), (16, 64, 33), (5, 64, 3000)])
def test_copy_of_blocks(gpu_device, heads, dim, blocks):
    from solution.kernels.attention import hip_block_cache_copy

    cache = _filled_cache(gpu_device, 1, heads, dim, BF16, blocks, [[0]], 71)
    before = {name: getattr(cache, name).clone() for name in _CODES}
    generator = _generator(72)
    origins = [-1] * blocks
    order = torch.randperm(blocks, generator=generator).tolist()
    third = blocks // 3
    for target in order[:third]:
        origins[target] = order[third + int(torch.randint(0, blocks - third, (1,), generator=generator))]
    origins[order[third]] = order[third]  # itself
    origins[order[-1]] = blocks  # no place
    origins[order[-2]] = -9
    want = [o if o >= 0 and o < blocks else t for t, o in enumerate(origins)]
    assert hip_block_cache_copy(cache, _words(origins, gpu_device)) == "hip_block_cache_copy"
    for name, held in before.items():
        assert torch.equal(getattr(cache, name), held[want]), name


def test_copy_leaves_out_blocks_whose_origin_is_written(gpu_device):
    from solution.kernels.attention import hip_block_cache_copy

    cache = _filled_cache(gpu_device, 1, 4, 64, F16, 8, [[0]], 73)
    before = {name: getattr(cache, name).clone() for name in _CODES}
    # 0 <- 1 <- 2: the first is left out; 3 and 4 would change places; 6 <- 5 and 7 <- 5 are copies
    hip_block_cache_copy(cache, _words([1, 2, -1, 4, 3, -1, 5, 5], gpu_device))
    for name, held in before.items():
        assert torch.equal(getattr(cache, name), held[[0, 2, 2, 3, 4, 5, 5, 5]]), name


def test_copy_of_more_than_four_gigabytes(gpu_device):
    from solution.kernels.attention import hip_block_cache_copy

    blocks = 36_000  # 65536 bytes of keys each
    cache = _filled_cache(gpu_device, 1, 16, 64, BF16, blocks, [[0]], 74)
    assert cache.key_codes.numel() > 2**31
    origins = torch.full((blocks,), -1, dtype=torch.int32, device=gpu_device)
    origins[0], origins[blocks - 1], origins[35_000] = blocks - 2, 1, 34_999
    want = [(0, blocks - 2), (blocks - 1, 1), (35_000, 34_999), (3, 3)]
    held = {name: [getattr(cache, name)[o].clone() for _, o in want] for name in _CODES}
    hip_block_cache_copy(cache, origins)
    for name, parts in held.items():
        for (target, _), part in zip(want, parts):
            assert torch.equal(getattr(cache, name)[target], part), (name, target)


@pytest.mark.parametrize("heads,dim,blocks", [(16, 64, 4200), (3, 128, 6000), (1, 64, 40_000)])
def test_copy_of_blocks_of_a_cache_larger_than_the_caches(gpu_device, heads, dim, blocks):
    """Any plan over more than 256 MB of codes: some places from others, some from places of
    no cache, some from themselves, some left out as their origin is written."""

    from solution.kernels.attention import hip_block_cache_copy

    cache = _filled_cache(gpu_device, 1, heads, dim, F16, blocks, [[0]], 77)
    assert cache.key_codes.numel() + cache.value_codes.numel() > 256 << 20
    before = {name: getattr(cache, name).clone() for name in _CODES}
    generator = _generator(78)
    origins = torch.where(torch.rand(blocks, generator=generator) < 0.4,
                          torch.randint(-2, blocks + 2, (blocks,), generator=generator), -1)
    place = torch.arange(blocks)
    written = (origins >= 0) & (origins < blocks) & (origins != place)
    takes = written & ~written[origins.clamp(0, blocks - 1)]
    assert 0.1 * blocks < int(takes.sum()) < int(written.sum())
    want = torch.where(takes, origins, place).to(gpu_device)
    hip_block_cache_copy(cache, _words(origins.tolist(), gpu_device))
    for name, held in before.items():
        assert torch.equal(getattr(cache, name), held[want]), name


@pytest.mark.parametrize("batch", [1, 2, 5, 64, 65, 300, 1024])
@pytest.mark.parametrize("heads,dim", [(1, 64), (3, 128)])
def test_fork_of_the_tails(gpu_device, batch, heads, dim):
    from solution.kernels.attention import hip_block_cache_fork

    cache = _filled_cache(gpu_device, batch, heads, dim, F16, 1, [[0]] * batch, 75)
    for seed in range(2):
        before = [cache.key_tail.clone(), cache.value_tail.clone()]
        sources = torch.randint(-1, batch + 1, (batch,), generator=_generator(seed)).tolist()
        if batch > 3:
            sources[:3] = [1, 0, 2]
        assert hip_block_cache_fork(cache, _words(sources, gpu_device)) == "hip_block_cache_fork"
        want = [s if 0 <= s < batch else b for b, s in enumerate(sources)]
        for tail, held in zip((cache.key_tail, cache.value_tail), before):
            assert torch.equal(tail, held[want])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,dim", [(1, 64), (3, 128)])
def test_take_back(gpu_device, dtype, heads, dim):
    """What the tail takes is what the read-back of the block gives; other tails stay."""

    from solution.kernels.attention import hip_block_cache_read, hip_block_cache_take_back

    lengths = [300, 300, 300, 300, 256, 70, 64, 320, 200, 200, -3, 10_000, 130, 10_000]
    ends = [299, 200, 192, 1, 255, 70, 0, 65, 201, -1, 5, 9_999, 64 + 5, 9_983]
    batch = len(lengths)
    table = [[5 * b + j for j in range(5)] for b in range(batch)]
    table[7][1] = -1  # no place
    table[12][1] = 10**6
    cache = _filled_cache(gpu_device, batch, heads, dim, dtype, 5 * batch, table, 76)
    firsts = [max(e, 0) // 64 * 64 for e in ends]
    key, value, _ = hip_block_cache_read(cache, _words(firsts, gpu_device), _words([10_000] * batch, gpu_device), 64)
    before = [cache.key_tail.clone(), cache.value_tail.clone()]
    assert hip_block_cache_take_back(cache, _words(lengths, gpu_device), _words(ends, gpu_device)) == "hip_block_cache_take_back"
    for b, (length, end) in enumerate(zip(lengths, ends)):
        back = end >= 0 and end % 64 > 0 and end // 64 < length // 64
        want = (key[b], value[b].transpose(-2, -1)) if back else (before[0][b], before[1][b])
        if back and end // 64 >= 5:  # behind the table
            want = (torch.full_like(key[b], math.nan), torch.full_like(before[1][b], math.nan))
        assert back == (b in (1, 3, 4, 7, 12, 13)), b
        for tail, held in zip((cache.key_tail, cache.value_tail), want):
            assert torch.equal(tail[b].isnan(), held.isnan()), b
            assert torch.equal(tail[b].nan_to_num(0.5), held.nan_to_num(0.5)), b


def test_pool_and_cache_refusals(gpu_device):
    from solution.kernels.attention import (
        BlockCache, BlockPool, hip_block_cache_copy, hip_block_cache_fork, hip_block_cache_take_back, hip_block_pool_fork,
        hip_block_pool_release, hip_block_pool_reserve,
    )

    pool = BlockPool.allocate(2, max_tokens=256, num_blocks=9, device=gpu_device)
    cache = BlockCache.allocate(2, 2, 64, max_tokens=256, num_blocks=9, block_table=pool.block_table, device=gpu_device)
    words, origins = _words([0, 0], gpu_device), _words([-1] * 9, gpu_device)
    for bad in (words.long(), words[:1], words.cpu(), words[None], None, _words([0, 0, 0, 0], gpu_device)[::2]):
        for call in (
            lambda w: hip_block_pool_reserve(pool, w, 3),
            lambda w: hip_block_pool_release(pool, w),
            lambda w: hip_block_pool_fork(pool, w, words),
            lambda w: hip_block_pool_fork(pool, words, w),
            lambda w: hip_block_cache_fork(cache, w),
            lambda w: hip_block_cache_take_back(cache, w, words),
            lambda w: hip_block_cache_take_back(cache, words, w),
        ):
            with pytest.raises(RuntimeError, match="ineligible"):
                call(bad)
    for tokens in (-1, 2**31, 1.5, True):
        with pytest.raises(RuntimeError, match="ineligible"):
            hip_block_pool_reserve(pool, words, tokens)
    for bad in (origins.long(), origins[:8], origins.cpu(), words):
        with pytest.raises(RuntimeError, match="ineligible"):
            hip_block_cache_copy(cache, bad)
    many = BlockPool.allocate(1025, max_tokens=64, num_blocks=9, device=gpu_device)
    wide = torch.zeros(1025, dtype=torch.int32, device=gpu_device)
    with pytest.raises(RuntimeError, match="ineligible"):
        hip_block_pool_fork(many, wide, wide)


def test_calls_without_sequences(gpu_device):
    from solution.kernels.attention import (
        BlockCache, BlockPool, hip_block_cache_copy, hip_block_cache_fork, hip_block_cache_take_back, hip_block_pool_compact,
        hip_block_pool_fork, hip_block_pool_release, hip_block_pool_reserve,
    )

    none = torch.zeros(0, dtype=torch.int32, device=gpu_device)
    pool = BlockPool.allocate(0, max_tokens=256, num_blocks=0, device=gpu_device)
    cache = BlockCache.allocate(0, 2, 64, max_tokens=256, num_blocks=0, block_table=pool.block_table, device=gpu_device)
    assert hip_block_pool_reserve(pool, none, 70)[0].shape == (0,)
    hip_block_pool_release(pool, none)
    hip_block_pool_fork(pool, none, none)
    origins, used, _ = hip_block_pool_compact(pool)
    assert origins.shape == (0,) and used.tolist() == [0]
    hip_block_cache_copy(cache, origins)
    hip_block_cache_fork(cache, none)
    hip_block_cache_take_back(cache, none, none)


# ---------------------------------------------------------------------------
# together


class _Serving:
    """One layer and a head, for a batch with adapters: what a step with drafts runs."""

    def __init__(self, device, batch, *, heads=4, kv_heads=2, dim=64, vocab=333, max_tokens=512, num_blocks=None, seed=0):
        from solution.kernels.attention import BlockCache, BlockPool
        from solution.kernels.norm import rotary_table
        from solution.kernels.projection import LowRankAdapters, quantize_linear_w4

        self.device, self.batch, self.heads, self.kv_heads, self.dim = device, batch, heads, kv_heads, dim
        width, out = 256, (heads + 2 * kv_heads) * dim
        to = lambda t: t.to(device)  # noqa: E731
        self.embedding = to(_rand((vocab, width), seed, BF16))
        self.weight = quantize_linear_w4(to(_rand((out, width), seed + 1, BF16, width**-0.5)), 128)
        self.adapters = LowRankAdapters.pack([
            (to(_rand((r, width), seed + 2 + r, BF16, width**-0.5)), to(_rand((out, r), seed + 3 + r, BF16, r**-0.5)), 1.5)
            for r in (8, 20, 5)
        ])
        self.head = to(_rand((vocab, heads * dim), seed + 9, BF16, 4 * (heads * dim) ** -0.5))
        self.table = rotary_table(max_tokens + 64, dim, device=device)
        self.pool = BlockPool.allocate(batch, max_tokens=max_tokens, device=device,
                                       num_blocks=batch * (max_tokens // 64) if num_blocks is None else num_blocks)
        self.cache = BlockCache.allocate(batch, kv_heads, dim, max_tokens=max_tokens, num_blocks=self.pool.num_blocks,
                                         block_table=self.pool.block_table, device=device)
        self.indices = _words([i % 5 - 1 for i in range(batch)], device)

    def logits(self, tokens, starts, counts=None):
        """Logits [batch, seq, vocab] after each of the new tokens, which the cache takes."""

        from solution.kernels.attention import hip_block_cache_append, hip_block_cache_attention, hip_block_pool_reserve
        from solution.kernels.norm import hip_qk_norm_rotary
        from solution.kernels.projection import hip_linear_w4, hip_low_rank_adapters

        seq = tokens.shape[1]
        hip_block_pool_reserve(self.pool, starts, seq, counts)
        x = self.embedding[tokens]
        packed, _ = hip_linear_w4(x, self.weight)
        packed, _ = hip_low_rank_adapters(x, packed, self.adapters, self.indices, counts, out=packed)
        packed = packed.view(self.batch, seq, -1, self.dim)
        q, k, v = (t.transpose(1, 2) for t in packed.tensor_split((self.heads, self.heads + self.kv_heads), dim=2))
        q, k, _ = hip_qk_norm_rotary(q, k, None, None, self.table, starts)
        hip_block_cache_append(self.cache, k, v, starts, counts)
        context, _ = hip_block_cache_attention(q, self.cache, starts, counts)
        return (context.float() @ self.head.float().t()).to(BF16)

    def settle(self, lengths, ends):
        from solution.kernels.attention import hip_block_cache_take_back, hip_block_pool_release

        hip_block_cache_take_back(self.cache, lengths, ends)
        hip_block_pool_release(self.pool, ends)


def _held(cache, lengths):
    from solution.kernels.attention import hip_block_cache_read

    most = max(1, int(lengths.max()))
    return hip_block_cache_read(cache, torch.zeros_like(lengths), lengths, most)[:2]


def test_steps_with_drafts_across_blocks(gpu_device):
    """Greedy requests with drafts that stand in part answer what they answer token by
    token: over many steps, across the blocks' ends and back, with the pool's places in
    use again.  What the cache holds is checked against the tokens' own keys and values."""

    batch, vocab, drafts, steps = 6, 333, 5, 40
    drafted = _Serving(gpu_device, batch, vocab=vocab, num_blocks=36, seed=81)
    generator = _generator(82)
    with torch.inference_mode():
        from solution.kernels.sampling import hip_verify_draft

        prompt = torch.randint(0, vocab, (batch, 61), generator=generator).to(gpu_device)
        counts = _words([61, 3, 60, 58, 1, 33], gpu_device)
        starts = torch.zeros(batch, dtype=torch.int32, device=gpu_device)
        logits = drafted.logits(prompt, starts, counts)
        last = logits[torch.arange(batch, device=gpu_device), counts.long() - 1].float().argmax(-1)
        starts = counts.clone()
        history = [prompt[b, : int(counts[b])].tolist() + [int(last[b])] for b in range(batch)]
        zero = torch.zeros(batch, device=gpu_device)
        book = None
        for step in range(steps):
            draft = torch.randint(0, vocab, (batch, drafts), generator=generator).to(gpu_device)
            tokens = torch.cat([last[:, None], draft], dim=1)
            logits = drafted.logits(tokens, starts)
            # drafts that the target would have chosen, cut at a place of its own for each request
            wish = logits[:, :drafts].float().argmax(-1)
            cut = torch.randint(0, drafts + 1, (batch,), generator=generator).to(gpu_device)
            place = torch.arange(drafts, device=gpu_device)
            same = torch.where(place < cut[:, None], wish, (wish + 1) % vocab)
            answer, accepted, _ = hip_verify_draft(logits, same, torch.rand((batch, drafts + 1), device=gpu_device),
                                                   temperatures=zero)
            assert torch.equal(accepted, cut.int())
            assert torch.equal(answer.gather(1, cut[:, None])[:, 0], logits.float().argmax(-1).gather(1, cut[:, None])[:, 0])
            # the tokens that the cache took are the random ones: as many of them stay as stand
            lengths, ends = starts + drafts + 1, starts + 1 + accepted
            drafted.settle(lengths, ends)
            for b in range(batch):
                history[b] += draft[b, : int(accepted[b])].tolist() + [int(answer[b, int(accepted[b])])]
            last = answer.gather(1, accepted.long()[:, None])[:, 0]
            starts = ends
            book = drafted.pool
            named = book.block_table[book.block_table >= 0]
            assert named.numel() == named.unique().numel() and int(book.holders.sum()) == named.numel()
            assert named.numel() == int((starts // 64).sum())
            if int(starts.max()) > 400:
                break
        assert step > 10 and int(starts.min()) > 64

        # every token that stayed, through the same layer at once
        whole = _Serving(gpu_device, batch, vocab=vocab, seed=81)
        most = int(starts.max())
        tokens = torch.tensor([(h[:most] + [0] * most)[:most] for h in history], device=gpu_device)
        whole.logits(tokens, torch.zeros_like(starts), starts)
        got, want = _held(drafted.cache, starts), _held(whole.cache, starts)
    for mine, other in zip(got, want):
        for b in range(batch):
            n = int(starts[b])
            a, w = mine[b, :, :n].double().cpu(), other[b, :, :n].double().cpu()
            # a value is rounded to a code: off by half a step, 2^-4 of it, or 2^-10 of a scale
            # that is at most the block's largest over 224.  Taken back and coded anew it
            # stays, but for a code that another scale leaves without its last bits: twice
            # that on either side, which covers the two sides' own roundings to 16 bits too
            largest = torch.stack([t.abs().amax(dim=(1, 2)) for t in (a, w)]).amax(0)[:, None, None]
            bound = 4 * (2.0**-4 * torch.maximum(a.abs(), w.abs()) + 2.0**-10 * largest / 224)
            assert ((a - w).abs() <= bound).all(), b


@pytest.mark.parametrize("places", [1, 2, 3, 6])
def test_steps_of_a_pool_that_runs_out(gpu_device, places):
    """Steps that ask for more places than there are, with the tokens that each appends cut
    to those before the first block without one: what stood stays, finite and as the
    tokens' own keys and values, and sequences go on as long as no block must be complete."""

    from solution.kernels.attention import hip_block_pool_reserve
    from solution.kernels.sampling import hip_verify_draft

    batch, vocab, drafts = 5, 101, 7
    model = _Serving(gpu_device, batch, vocab=vocab, num_blocks=places, max_tokens=192, seed=94)
    generator = _generator(95)
    with torch.inference_mode():
        first = [60, 57, 63, 30, 100]
        prompt = torch.randint(0, vocab, (batch, 100), generator=generator).to(gpu_device)
        starts = _words(first, gpu_device)
        model.logits(prompt, torch.zeros_like(starts), starts)
        assert model.pool.block_table[4].tolist() == [0, -1, -1]
        history = [prompt[b, :n].tolist() for b, n in enumerate(first)]
        wanted = _words([8, 8, 8, 3, 8], gpu_device)
        short = 0
        for step in range(16):
            tokens = torch.randint(0, vocab, (batch, drafts + 1), generator=generator).to(gpu_device)
            missing, _ = hip_block_pool_reserve(model.pool, starts, drafts + 1, wanted)
            counts = torch.minimum(wanted, 64 * ((starts + wanted) // 64 + 1 - missing) - 1 - starts)
            logits = model.logits(tokens, starts, counts)
            same = logits[:, :drafts].float().argmax(-1)  # the first of them stand
            cut = torch.randint(0, drafts + 1, (batch, 1), generator=generator).to(gpu_device)
            same = torch.where(torch.arange(drafts, device=gpu_device) < cut, same, (same + 1) % vocab)
            zero = torch.zeros(batch, device=gpu_device)
            uniforms = torch.rand((batch, drafts + 1), device=gpu_device)
            answer, accepted, _ = hip_verify_draft(logits, same, uniforms, counts=counts - 1, temperatures=zero)
            assert torch.equal(accepted, torch.minimum(cut[:, 0], counts - 1).int())
            lengths, ends = starts + counts, starts + 1 + accepted
            model.settle(lengths, ends)
            for b, (start, end) in enumerate(zip(starts.tolist(), ends.tolist())):
                history[b] += tokens[b, : end - start].tolist()
                # a sequence waits only where its next token would complete a block without a place
                assert end > start or (start % 64 == 63 and int(missing[b]) > 0), (step, b)
            short += int((missing > 0).sum())
            starts = ends
            assert model.pool.block_table.ge(0).sum(1).tolist() == [n // 64 for n in starts.tolist()]
        assert short > 0
        whole = _Serving(gpu_device, batch, vocab=vocab, max_tokens=192, seed=94)
        most = int(starts.max())
        tokens = torch.tensor([h + [0] * (most - len(h)) for h in history], device=gpu_device)
        whole.logits(tokens, torch.zeros_like(starts), starts)
        got, want = _held(model.cache, starts), _held(whole.cache, starts)
    for mine, other in zip(got, want):
        for b, n in enumerate(starts.tolist()):
            a, w = mine[b, :, :n].double().cpu(), other[b, :, :n].double().cpu()
            # as in test_steps_with_drafts_across_blocks: two codings on either side
            largest = torch.stack([t.abs().amax(dim=(1, 2)) for t in (a, w)]).amax(0)[:, None, None]
            bound = 4 * (2.0**-4 * torch.maximum(a.abs(), w.abs()) + 2.0**-10 * largest / 224)
            assert a.isfinite().all() and ((a - w).abs() <= bound).all(), b


def test_beams_share_blocks_and_part(gpu_device):
    """Forked sequences hold what their sources held, then their own tokens; the
    sources' stay as they were; after compaction all of it stands at lower places."""

    from solution.kernels.attention import (
        hip_block_cache_copy, hip_block_cache_fork, hip_block_pool_compact, hip_block_pool_fork, hip_block_pool_release,
    )

    batch, vocab = 6, 211
    model = _Serving(gpu_device, batch, vocab=vocab, num_blocks=48, seed=83)
    generator = _generator(84)
    with torch.inference_mode():
        prompt = torch.randint(0, vocab, (batch, 200), generator=generator).to(gpu_device)
        lengths = _words([200, 130, 64, 190, 5, 128], gpu_device)
        model.logits(prompt, torch.zeros_like(lengths), lengths)
        before = _held(model.cache, lengths)
        sources = _words([3, 0, 0, 5, -1, 0], gpu_device)
        hip_block_pool_fork(model.pool, sources, lengths)
        hip_block_cache_fork(model.cache, sources)
        origin = torch.tensor([3, 0, 0, 5, 4, 0], device=gpu_device)
        lengths = lengths[origin]
        assert lengths.tolist() == [190, 200, 200, 128, 5, 200]
        for mine, held in zip(_held(model.cache, lengths), before):
            assert torch.equal(mine, held[origin])
        assert int((model.pool.holders > 0).sum()) == 2 + 3 + 2  # of 190, 200 and 128 tokens
        # each goes on with tokens of its own, across the end of a block
        model.logits(torch.randint(0, vocab, (batch, 77), generator=generator).to(gpu_device), lengths)
        longer = lengths + 77
        grown = _held(model.cache, longer)
        for mine, held in zip(grown, before):
            for b in range(batch):
                whole = int(lengths[b]) // 64 * 64
                assert torch.equal(mine[b, :, :whole], held[origin[b], :, :whole])
        assert not torch.equal(grown[0][1, :, 200:], grown[0][2, :, 200:])
        # two have ended; the rest move to the lowest places
        ended = _words([-1, 0, -1, -1, 0, -1], gpu_device)
        hip_block_pool_release(model.pool, ended)
        origins, used, _ = hip_block_pool_compact(model.pool)
        hip_block_cache_copy(model.cache, origins)
        stay = torch.tensor([0, 2, 3, 5], device=gpu_device)
        assert int((origins >= 0).sum()) > 0
        assert int(model.pool.block_table.max()) < int(used) == int((model.pool.holders > 0).sum())
        after = _held(model.cache, longer)
        for mine, held in zip(after, grown):
            assert torch.equal(mine[stay], held[stay])


def test_captured_steps_replay_as_eager_ones(gpu_device):
    """A whole step with drafts in one graph, replayed beside eager work: reserve, adapters,
    append, attention, verification, taking back and release, on positions that move."""

    from solution.kernels.sampling import hip_verify_draft

    batch, vocab, drafts = 4, 97, 3
    models = [_Serving(gpu_device, batch, vocab=vocab, num_blocks=40, seed=85) for _ in range(2)]
    generator = _generator(86)

    def step(model, tokens, uniforms, starts):
        logits = model.logits(tokens, starts)
        answer, accepted, _ = hip_verify_draft(logits, tokens[:, 1:].contiguous(), uniforms)
        ends = starts + 1 + accepted
        model.settle(starts + drafts + 1, ends)
        return answer, accepted, ends

    with torch.inference_mode():
        prompt = torch.randint(0, vocab, (batch, 62), generator=generator).to(gpu_device)
        zeros = torch.zeros(batch, dtype=torch.int32, device=gpu_device)
        for model in models:
            model.logits(prompt, zeros)
        first = torch.full((batch,), 62, dtype=torch.int32, device=gpu_device)
        tokens = torch.randint(0, vocab, (batch, drafts + 1), generator=generator).to(gpu_device)
        uniforms = torch.rand((batch, drafts + 1), generator=generator).to(gpu_device)
        starts = first.clone()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            answer, accepted, ends = step(models[0], tokens, uniforms, starts)
            starts.copy_(ends)
        torch.cuda.current_stream().wait_stream(stream)
        eager = first.clone()
        for i in range(12):
            fresh = torch.randint(0, vocab, (batch, drafts + 1), generator=generator).to(gpu_device)
            chance = torch.rand((batch, drafts + 1), generator=generator).to(gpu_device) * (0.05 if i % 2 else 1.0)
            want = step(models[1], fresh, chance, eager)
            eager = want[2]
            tokens.copy_(fresh), uniforms.copy_(chance)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(answer, want[0]) and torch.equal(accepted, want[1]) and torch.equal(starts, eager), i
    assert torch.equal(models[0].pool.block_table, models[1].pool.block_table)
    assert torch.equal(models[0].pool.holders, models[1].pool.holders)
    for name in _CODES + ("key_tail", "value_tail"):
        assert torch.equal(getattr(models[0].cache, name), getattr(models[1].cache, name)), name


@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("batch,vocab", [(4, 9001), (70, 4097), (600, 203)])
def test_captured_verification_of_few_and_many_requests(gpu_device, batch, vocab, sampled):
    """Two, three and four launches of a graph, replayed on other inputs beside eager calls."""

    from solution.kernels.sampling import hip_verify_draft

    drafts = 3
    generator = _generator(101)

    def inputs(seed):
        made = [t.to(gpu_device) for t in _drafted(batch, drafts, vocab, BF16, seed, near=0.2)]
        made.append(torch.randint(-1, drafts + 2, (batch,), generator=generator).int().to(gpu_device))
        heat = torch.tensor([1.0, 0.0, 0.5])[torch.randint(0, 3, (batch,), generator=generator)]
        return made + [heat.to(gpu_device)]

    def call(target, draft, tokens, uniforms, counts, temperatures):
        return hip_verify_draft(target, tokens, uniforms, draft if sampled else None, counts=counts, temperatures=temperatures)[:2]

    with torch.inference_mode():
        held = inputs(102)
        call(*held)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = call(*held)
        answers = set()
        for i in range(5):
            fresh = inputs(103 + i)
            want = call(*fresh)
            for mine, other in zip(held, fresh):
                mine.copy_(other)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(captured[0], want[0]) and torch.equal(captured[1], want[1]), i
            answers |= set(captured[1].tolist())
        assert len(answers) > (2 if sampled else 1)  # (a certain draft of many tokens seldom stands)


@pytest.mark.parametrize("batch,width,blocks", [(6, 9, 60), (40, 30, 20_000)])
def test_captured_forks_and_compactions_replay_as_eager_ones(gpu_device, batch, width, blocks):
    """Reserve, fork, release, compaction and copy in one graph, on sources and lengths that
    change; pools compacted in one launch and in two."""

    from solution.kernels.attention import (
        BlockPool, hip_block_cache_copy, hip_block_cache_fork, hip_block_pool_compact, hip_block_pool_fork,
        hip_block_pool_release, hip_block_pool_reserve,
    )

    tokens = 130
    caches = [_filled_cache(gpu_device, batch, 2, 64, BF16, blocks, [[-1] * width] * batch, 104) for _ in range(2)]
    pools = [BlockPool(c.block_table, torch.zeros(blocks, dtype=torch.int32, device=gpu_device)) for c in caches]
    for pool in pools:  # some places are someone else's, so that there is something to move
        pool.holders[::3] = 1
    generator = _generator(105)

    def step(pool, cache, starts, sources, lengths, ends):
        missing = hip_block_pool_reserve(pool, starts, tokens)[0]
        hip_block_pool_fork(pool, sources, lengths)
        hip_block_cache_fork(cache, sources)
        hip_block_pool_release(pool, ends)
        origins, used, _ = hip_block_pool_compact(pool)
        hip_block_cache_copy(cache, origins)
        return missing, origins, used

    with torch.inference_mode():
        static = [torch.zeros(batch, dtype=torch.int32, device=gpu_device) for _ in range(4)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step(pools[0], caches[0], *static)
        starts, moved = torch.zeros(batch, dtype=torch.int64), 0
        for i in range(8):
            sources = torch.randint(-1, batch + 1, (batch,), generator=generator)
            lengths = starts + tokens
            origin = torch.where((sources >= 0) & (sources < batch), sources, torch.arange(batch))
            ends = (lengths[origin] - torch.randint(0, 150, (batch,), generator=generator)).clamp(min=0)
            ends[torch.rand(batch, generator=generator) < 0.1] = 0
            given = [_words(t.tolist(), gpu_device) for t in (starts, sources, lengths, ends)]
            want = step(pools[1], caches[1], *given)
            for mine, other in zip(static, given):
                mine.copy_(other)
            graph.replay()
            torch.cuda.synchronize()
            for mine, other in zip(captured, want):
                assert torch.equal(mine, other), i
            assert torch.equal(pools[0].block_table, pools[1].block_table), i
            assert torch.equal(pools[0].holders, pools[1].holders), i
            for name in _CODES + ("key_tail", "value_tail"):
                assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), (i, name)
            moved += int((want[1] >= 0).sum())
            starts = ends
        assert moved > 0


def test_two_streams_at_once(gpu_device):
    """Calls that overlap on two streams have workspaces of their own."""

    from solution.kernels.projection import LowRankAdapters, hip_low_rank_adapters
    from solution.kernels.sampling import hip_verify_draft

    drafts = [[t.to(gpu_device) for t in _drafted(16, 4, 30_000, BF16, 87 + i)] for i in range(2)]
    packed = LowRankAdapters(*(t.to(gpu_device) for t in _adapter_tensors(4, 32, 1024, 2048, BF16, 89)))
    rows = [(_rand((16, 1024), 90 + i, BF16).to(gpu_device), _rand((16, 2048), 92 + i, BF16).to(gpu_device)) for i in range(2)]
    indices = _words([i % 4 for i in range(16)], gpu_device)

    def work(i):
        target, draft, tokens, uniforms = drafts[i]
        return (*hip_verify_draft(target, tokens, uniforms, draft)[:2], hip_low_rank_adapters(*rows[i], packed, indices)[0])

    with torch.inference_mode():
        want = [work(i) for i in range(2)]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = [[], []]
        for _ in range(6):
            for i, stream in enumerate(streams):
                with torch.cuda.stream(stream):
                    got[i].append(work(i))
        torch.cuda.synchronize()
    for w, outs in zip(want, got):
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(w, out))

"""The decoding operators without a GPU: refusals of the C entries before any
launch, eligibility in Python, the cache's and the packed weight's own checks, and
the 4-bit format against a plain decoder."""

from __future__ import annotations

import importlib
import re
from pathlib import Path

import pytest
import torch

from solution.kernels.attention import (
    BlockCache,
    can_use_hip_block_cache_append,
    can_use_hip_block_cache_attention,
    hip_block_cache_append,
    hip_block_cache_attention,
    hip_block_cache_read,
)
from solution.kernels.hip import _library
from solution.kernels.norm import can_use_hip_qk_norm_rotary, hip_qk_norm_rotary, rotary_table
from solution.kernels.projection import (
    PackedLinearW4,
    can_use_hip_linear_w4,
    hip_linear_w4,
    pack_linear_w4_codes,
    quantize_linear_w4,
)

# An address that the host checks may look at and no kernel reads: every call below
# is refused, or has nothing to do, before a launch.
P = 0x10000
BF16, F16, F32 = 2, 1, 0
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 4


def _call(name, defaults, **changes):
    unknown = set(changes) - set(defaults)
    assert not unknown, unknown
    return getattr(_library.load_library(), name)(*{**defaults, **changes}.values())


ROTARY = dict(
    query=P, key=P, query_weight=P, query_bias=None, key_weight=P, key_bias=None, table=P, starts=P, query_out=P,
    key_out=P, batch=1, seq_len=4, heads=8, kv_heads=2, head_dim=64, q_sb=0, q_sh=64, q_ss=640, k_sb=0, k_sh=64,
    k_ss=640, rotary_dim=64, table_rows=10, interleaved=0, norm_kind=1, eps=1e-6, dtype=BF16, param_dtype=F32,
    stream=None,
)


@pytest.mark.parametrize(
    "changes,status",
    [
        ({"batch": 0}, OK),
        ({"seq_len": 0}, OK),
        ({"head_dim": 96}, UNSUPPORTED),
        ({"dtype": 7}, INVALID),
        ({"param_dtype": F16}, UNSUPPORTED),
        ({"norm_kind": 2}, INVALID),
        ({"eps": -1.0}, INVALID),
        ({"eps": float("nan")}, INVALID),
        ({"heads": 0}, INVALID),
        ({"kv_heads": -1}, INVALID),
        ({"batch": -1}, INVALID),
        ({"batch": 1 << 16, "seq_len": 1 << 15}, UNSUPPORTED),
        ({"rotary_dim": 128}, UNSUPPORTED),
        ({"rotary_dim": 24}, UNSUPPORTED),
        ({"rotary_dim": 12, "interleaved": 1}, UNSUPPORTED),
        ({"rotary_dim": -16}, UNSUPPORTED),
        ({"query": None}, INVALID),
        ({"key_out": None}, INVALID),
        ({"table": None}, INVALID),
        ({"table_rows": -1}, INVALID),
        ({"key": P + 8}, INVALID),
        ({"query_weight": P + 4}, INVALID),
        ({"starts": P + 2}, INVALID),
        ({"q_ss": 641}, INVALID),
        ({"k_sh": 4}, INVALID),
    ],
)
def test_rotary_entry_refuses_before_launch(changes, status):
    assert _call("sah_qk_norm_rotary", ROTARY, **changes) == status


CACHE = dict(key_codes=P, value_codes=P, key_scales=P, value_scales=P, key_tail=P, value_tail=P, table=P)
APPEND = dict(
    key=P, value=P, **CACHE, starts=P, counts=None, batch=2, kv_heads=2, seq_len=3, head_dim=64, k_sb=0, k_sh=64,
    k_ss=256, v_sb=0, v_sh=64, v_ss=256, num_blocks=4, max_blocks=2, dtype=BF16, stream=None,
)
READ = dict(
    **CACHE, firsts=P, lengths=P, key=P, value=P, batch=2, kv_heads=2, tokens=3, head_dim=64, num_blocks=4,
    max_blocks=2, dtype=BF16, stream=None,
)
ATTENTION = dict(
    query=P, **CACHE, starts=P, counts=None, output=P, batch=2, heads=4, kv_heads=2, seq_len=1, head_dim=64,
    q_sb=0, q_sh=64, q_ss=256, o_sb=256, o_ss=256, num_blocks=4, max_blocks=2, max_length=128, scale=0.125,
    dtype=BF16, workspace=None, workspace_bytes=0, stream=None,
)
OF_CACHE = [
    ({"batch": 0}, OK),
    ({"head_dim": 96}, UNSUPPORTED),
    ({"dtype": F32}, UNSUPPORTED),
    ({"batch": -1}, INVALID),
    ({"kv_heads": 0}, INVALID),
    ({"num_blocks": -1}, INVALID),
    ({"max_blocks": -1}, INVALID),
    ({"max_blocks": 1 << 30}, INVALID),
    ({"key_codes": None}, INVALID),
    ({"value_scales": None}, INVALID),
    ({"table": None}, INVALID),
    ({"value_tail": None}, INVALID),
    ({"key_tail": P + 8}, INVALID),
    ({"value_codes": P + 1}, INVALID),
    ({"key_scales": P + 2}, INVALID),
]


@pytest.mark.parametrize(
    "changes,status",
    OF_CACHE
    + [
        ({"seq_len": 0}, OK),
        ({"seq_len": -1}, INVALID),
        ({"key": None}, INVALID),
        ({"starts": None}, INVALID),
        ({"value": P + 8}, INVALID),
        ({"counts": P + 1}, INVALID),
        ({"v_ss": 100}, INVALID),
        ({"batch": 1 << 20, "seq_len": 1 << 20}, UNSUPPORTED),
    ],
)
def test_append_entry_refuses_before_launch(changes, status):
    assert _call("sah_block_cache_append", APPEND, **changes) == status


@pytest.mark.parametrize(
    "changes,status",
    OF_CACHE
    + [
        ({"tokens": 0}, OK),
        ({"tokens": -1}, INVALID),
        ({"lengths": None}, INVALID),
        ({"value": None}, INVALID),
        ({"key": P + 2}, INVALID),
        ({"firsts": P + 2}, INVALID),
        ({"batch": 1 << 20, "tokens": 1 << 20}, UNSUPPORTED),
    ],
)
def test_read_entry_refuses_before_launch(changes, status):
    assert _call("sah_block_cache_read", READ, **changes) == status


@pytest.mark.parametrize(
    "changes,status",
    OF_CACHE
    + [
        ({"seq_len": 0}, OK),
        ({"seq_len": -1}, INVALID),
        ({"heads": 5}, INVALID),
        ({"heads": 0}, INVALID),
        ({"scale": float("nan")}, INVALID),
        ({"scale": float("inf")}, INVALID),
        ({"scale": 3e38}, INVALID),
        ({"max_length": -1}, INVALID),
        ({"output": None}, INVALID),
        ({"query": P + 8}, INVALID),
        ({"q_ss": 4}, INVALID),
        ({"o_sb": 4}, INVALID),
        ({"starts": P + 1}, INVALID),
        # a history long enough to be split, with no or too little workspace
        ({"max_length": 100000}, WORKSPACE),
        ({"max_length": 100000, "workspace": P, "workspace_bytes": 64}, WORKSPACE),
        ({"max_length": 100000, "workspace": P + 4, "workspace_bytes": 1 << 30}, INVALID),
    ],
)
def test_attention_entry_refuses_before_launch(changes, status):
    assert _call("sah_block_cache_attention", ATTENTION, **changes) == status


def test_attention_workspace_sizes():
    size = _library.load_library().sah_block_cache_attention_workspace_bytes
    assert size(1, 1, 16, 16, 64, 64) == 0
    assert size(1, 0, 16, 16, 64, 100000) == 0
    assert size(0, 1, 16, 16, 64, 100000) == 0
    assert size(1, 1, 16, 3, 64, 100000) == 0  # not a size that runs
    split = size(1, 1, 16, 16, 64, 100000)
    assert split > 0 and split % (16 * (64 + 2) * 4) == 0


LINEAR = dict(
    x=P, codes=P, scales=P, bias=None, y=P, rows=4, in_features=256, out_features=32, group_size=64, x_stride=256,
    y_stride=32, dtype=BF16, activation=0, stream=None,
)


@pytest.mark.parametrize(
    "changes,status",
    [
        ({"rows": 0}, OK),
        ({"rows": -1}, INVALID),
        ({"dtype": F32}, UNSUPPORTED),
        ({"activation": 2}, UNSUPPORTED),
        ({"group_size": 16}, UNSUPPORTED),
        ({"in_features": 192}, UNSUPPORTED),
        ({"out_features": 24}, UNSUPPORTED),
        ({"in_features": 0}, INVALID),
        ({"codes": None}, INVALID),
        ({"x": P + 8}, INVALID),
        ({"bias": P + 4}, INVALID),
        ({"x_stride": 257}, INVALID),
        ({"y_stride": 36}, INVALID),
        ({"rows": 1 << 39}, UNSUPPORTED),
        ({"x_stride": -256}, UNSUPPORTED),
        ({"x_stride": 2**25 + 8}, UNSUPPORTED),
    ],
)
def test_linear_w4_entry_refuses_before_launch(changes, status):
    assert _call("sah_linear_w4", LINEAR, **changes) == status


@pytest.mark.parametrize("changes,status", [({"y_stride": 24}, INVALID), ({"y_stride": 0}, INVALID), ({"y_stride": -32}, INVALID),
                                            ({"rows": 0, "y_stride": 0}, OK)])
def test_linear_w4_entry_refuses_rows_of_y_that_overlap(changes, status):
    assert _call("sah_linear_w4", LINEAR, **changes) == status


@pytest.mark.parametrize(
    "shape,strides,want",
    [
        ((128,), (1,), 128),
        ((3, 128), (136, 1), 136),
        ((3, 128), (0, 1), 0),
        ((1, 128), (2**26, 1), 128),
        ((2, 128), (2**25, 1), 2**25),
        ((2, 128), (2**25 + 8, 1), None),
        ((2, 128), (132, 1), None),
        ((2, 128), (128, 2), None),
        ((2, 3, 128), (384, 128, 1), 128),
        ((2, 3, 128), (512, 128, 1), None),
        ((2, 1, 128), (512, 7, 1), 512),
    ],
)
def test_linear_w4_rows_at_one_stride(shape, strides, want):
    module = importlib.import_module("solution.kernels.projection.hip_linear_w4")
    assert module._row_stride(shape, strides) == want


def _cpu_cache(**changes):
    sizes = dict(dtype=torch.bfloat16, device="cpu", max_tokens=200)
    return BlockCache.allocate(2, 3, 64, **{**sizes, **changes})


def test_cache_allocation():
    cache = _cpu_cache()
    assert cache.batch == 2 and cache.kv_heads == 3 and cache.head_dim == 64
    assert cache.block_table.tolist() == [[0, 1, 2], [3, 4, 5]] and cache.max_tokens == 255
    shared = _cpu_cache(num_blocks=10, block_table=cache.block_table)
    assert shared.key_codes.shape == (10, 3, 64, 64) and shared.block_table is cache.block_table
    assert _cpu_cache(num_blocks=4).block_table.eq(-1).all()
    short = _cpu_cache(max_tokens=63)
    assert short.block_table.shape == (2, 0) and short.key_codes.shape[0] == 0 and short.max_tokens == 63


@pytest.mark.parametrize(
    "name,make",
    [
        ("key_codes", lambda t: t.to(torch.int8)),
        ("value_codes", lambda t: t[:, :, :, :32]),
        ("key_scales", lambda t: t.double()),
        ("value_scales", lambda t: t[:-1]),
        ("key_tail", lambda t: t.float()),
        ("value_tail", lambda t: t.half()),
        ("value_tail", lambda t: t.transpose(-2, -1)),
        ("block_table", lambda t: t.long()),
        ("block_table", lambda t: t[0]),
        ("key_tail", lambda t: t[..., :32]),
    ],
)
def test_cache_of_tensors_that_do_not_belong_together(name, make):
    cache = _cpu_cache()
    parts = {field: getattr(cache, field) for field in cache.__dataclass_fields__}
    BlockCache(**parts)
    parts[name] = make(parts[name])
    with pytest.raises(ValueError):
        BlockCache(**parts)


def test_operators_refuse_cpu_tensors():
    cache = _cpu_cache()
    starts = torch.zeros(2, dtype=torch.int32)
    kv = torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="ineligible"):
        hip_block_cache_append(cache, kv, kv, starts)
    with pytest.raises(RuntimeError, match="ineligible"):
        hip_block_cache_read(cache, starts, starts, 4)
    with pytest.raises(RuntimeError, match="ineligible"):
        hip_block_cache_attention(kv, cache, starts)
    with pytest.raises(RuntimeError, match="ineligible"):
        hip_qk_norm_rotary(kv, kv, None, None, rotary_table(4, 64, device="cpu"), starts)
    packed = quantize_linear_w4(torch.ones(16, 128, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="ineligible"):
        hip_linear_w4(torch.zeros(1, 128, dtype=torch.bfloat16), packed)


def test_rotary_table():
    table = rotary_table(1001, 16, base=500.0, device="cpu")
    assert table.shape == (1001, 16) and table.dtype == torch.float32
    angle = 1000 * 500.0 ** (-torch.arange(8, dtype=torch.float64) / 8)
    assert torch.equal(table[1000], torch.cat([angle.cos(), angle.sin()]).float())
    for bad in ((-1, 16), (4, 7), (4, 0)):
        with pytest.raises(ValueError):
            rotary_table(*bad, device="cpu")


def _decoded(word):
    """The eight codes of a word, bit by bit."""

    word &= 0xFFFFFFFF
    codes = []
    for e in range(8):
        turned = word if e < 4 else ((word >> 4) | (word << 28)) & 0xFFFFFFFF
        byte = (turned >> (8 * (e % 4))) & 0xFF
        codes.append((byte & 7) * (-1 if byte & 0x80 else 1))
    return codes


@pytest.mark.parametrize("group", [32, 64, 128])
def test_packed_words_hold_the_codes(group):
    generator = torch.Generator().manual_seed(group)
    out_features, in_features = 48, 384
    codes = torch.randint(-7, 8, (out_features, in_features), generator=generator)
    scales = torch.rand(out_features, in_features // group, generator=generator).to(torch.float16)
    packed = pack_linear_w4_codes(codes, scales)
    assert packed.group_size == group and packed.out_features == out_features and packed.in_features == in_features
    for n, k, lane, step in ((0, 0, 0, 0), (2, 1, 37, 3), (1, 2, 63, 1), (0, 2, 16, 2)):
        first = 128 * k + 32 * step + 8 * (lane // 16)
        want = codes[16 * n + lane % 16, first : first + 8].tolist()
        assert _decoded(int(packed.codes[n, k, lane, step])) == want
    want = codes.float() * scales.float().repeat_interleave(group, dim=1)
    assert torch.equal(packed.dequantize(), want)


def test_quantized_weights_are_within_half_a_step():
    generator = torch.Generator().manual_seed(3)
    weight = torch.randn(32, 256, generator=generator).to(torch.bfloat16)
    weight[5, 64:128] = 0.0
    packed = quantize_linear_w4(weight, 64)
    scales = packed.scales.t().float().repeat_interleave(64, dim=1)
    # half a step, and what the scale's rounding (2^-8 of seven steps) takes off the largest codes
    bound = scales * (0.5 + 7 * 2.0**-8)
    assert bool(((packed.dequantize() - weight.float()).abs() <= bound).all())
    assert bool((packed.dequantize()[5, 64:128] == 0).all())


@pytest.mark.parametrize(
    "make",
    [
        lambda: pack_linear_w4_codes(torch.full((16, 128), 8), torch.ones(16, 1).half()),
        lambda: pack_linear_w4_codes(torch.full((16, 128), -8), torch.ones(16, 1).half()),
        lambda: pack_linear_w4_codes(torch.zeros(16, 128), torch.ones(16, 1).half()),
        lambda: pack_linear_w4_codes(torch.zeros(8, 128, dtype=torch.int8), torch.ones(8, 1).half()),
        lambda: pack_linear_w4_codes(torch.zeros(16, 96, dtype=torch.int8), torch.ones(16, 3).half()),
        lambda: pack_linear_w4_codes(torch.zeros(16, 128, dtype=torch.int8), torch.ones(32, 1).half()),
        lambda: pack_linear_w4_codes(torch.zeros(16, 128, dtype=torch.int8), torch.ones(16, 8).half()),
        lambda: pack_linear_w4_codes(torch.zeros(16, 128, dtype=torch.int8), torch.ones(16, 1)),
        lambda: quantize_linear_w4(torch.ones(16, 128)),
        lambda: quantize_linear_w4(torch.ones(16, 128).half(), 16),
        lambda: quantize_linear_w4(torch.full((16, 128), float("inf")).half()),
        lambda: PackedLinearW4(torch.zeros(1, 1, 64, 4), torch.ones(1, 16).half()),
        lambda: PackedLinearW4(torch.zeros(1, 0, 64, 4, dtype=torch.int32), torch.ones(1, 16).half()),
    ],
)
def test_weights_that_cannot_be_packed(make):
    with pytest.raises(ValueError):
        make()


@pytest.fixture
def without_a_gpu(monkeypatch):
    """The operators' eligibility checks on CPU tensors: everything but the device."""

    for name in ("attention.hip_block_cache", "norm.hip_qk_rotary", "projection.hip_linear_w4"):
        monkeypatch.setattr(importlib.import_module(f"solution.kernels.{name}"), "library_for", lambda index: object())


def _requests():
    """For each operator its check, the arguments of a call that it takes, and those that may be differentiated."""

    cache = _cpu_cache()
    starts = torch.zeros(2, dtype=torch.int32)
    kv = torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16)
    weight, bias = torch.ones(64), torch.zeros(64)
    packed = quantize_linear_w4(torch.ones(16, 128, dtype=torch.bfloat16))
    x, b = torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(16, dtype=torch.bfloat16)
    return {
        "append": (can_use_hip_block_cache_append, dict(cache=cache, key=kv, value=kv, starts=starts), ("key", "value")),
        "attention": (can_use_hip_block_cache_attention, dict(query=kv, cache=cache, starts=starts), ("query",)),
        "rotary": (
            can_use_hip_qk_norm_rotary,
            dict(query=kv, key=kv, query_weight=weight, key_weight=weight, table=rotary_table(4, 64, device="cpu"),
                 starts=starts, query_bias=bias, key_bias=bias),
            ("query", "key", "query_weight", "key_weight", "query_bias", "key_bias", "table"),
        ),
        "linear": (can_use_hip_linear_w4, dict(value=x, weight=packed, bias=b), ("value", "bias")),
    }


@pytest.mark.parametrize("operator", ["append", "attention", "rotary", "linear"])
def test_inputs_with_tangents_are_refused(without_a_gpu, operator):
    """A dual tensor asks for no gradient and keeps its tangent under no_grad: answering
    without the tangent would drop it."""

    check, arguments, names = _requests()[operator]
    assert check(**arguments)
    with torch.no_grad(), torch.autograd.forward_ad.dual_level():
        assert check(**arguments)
        for name in names:
            value = arguments[name]
            dual = torch.autograd.forward_ad.make_dual(value, torch.ones_like(value))
            assert not check(**{**arguments, name: dual}), name
    with torch.no_grad():
        assert check(**arguments)


def test_caches_and_weights_with_tangents_are_refused():
    cache, packed = _cpu_cache(), quantize_linear_w4(torch.ones(16, 128, dtype=torch.bfloat16))
    parts = {field: getattr(cache, field) for field in cache.__dataclass_fields__}
    with torch.autograd.forward_ad.dual_level():
        make_dual = torch.autograd.forward_ad.make_dual
        for name in ("key_scales", "value_tail"):
            with pytest.raises(ValueError):
                BlockCache(**{**parts, name: make_dual(parts[name], torch.ones_like(parts[name]))})
        with pytest.raises(ValueError):
            PackedLinearW4(packed.codes, make_dual(packed.scales, torch.ones_like(packed.scales)))


@pytest.mark.parametrize("scale,taken", [(0.0, True), (-3.0, True), (2.0**127, True), (1e39, False), (3e38, False),
                                         (-1e39, False), (float("inf"), False), (float("nan"), False)])
def test_scales_that_the_attention_takes(without_a_gpu, scale, taken):
    check, arguments, _ = _requests()["attention"]
    assert check(**arguments, scale=scale) is taken
    if taken:  # the C entry takes it too (of a batch of none, for which nothing is launched)
        assert _call("sah_block_cache_attention", ATTENTION, scale=scale, batch=0) == OK


def _parameters(entry):
    """A C entry's parameter names, from the header."""

    header = (Path(__file__).resolve().parents[1] / "include" / "shape_aware_hip.h").read_text()
    declared = re.search(rf"\b{entry}\((.*?)\);", re.sub(r"/\*.*?\*/", "", header, flags=re.S), flags=re.S)[1]
    return [re.findall(r"\w+", parameter)[-1] for parameter in declared.split(",")]


def _example(entry, values):
    """The documented call of ``entry``: its arguments by name, numbers evaluated."""

    text = (Path(__file__).resolve().parents[1] / "INTEGRATION.md").read_text()
    call = re.search(rf"rc = {entry}\((.*?)\);", re.sub(r"/\*.*?\*/", "", text, flags=re.S), flags=re.S)[1]
    arguments = [part.strip() for part in call.replace("(sah_stream_t)", "").split(",")]
    names = _parameters(entry)
    assert len(arguments) == len(names)
    number = lambda text: eval(text, {}, values) if re.fullmatch(r"[\w +*()]*\w[\w +*()]*", text) else text  # noqa: E731
    known = lambda text: all(w.isdigit() or w in values for w in re.findall(r"\w+", text))  # noqa: E731
    return {name: number(text) if known(text) else text for name, text in zip(names, arguments)}


def test_the_documented_step_stays_in_its_tensors():
    """The C example's strides reach the last element of each tensor, and not beyond."""

    sizes = dict(B=3, S=5, H=6, Hkv=2, D=256, N=(6 + 2 * 2) * 64, num_blocks=9, max_blocks=4, max_length=300, table_rows=400)
    batch, seq, heads, kv_heads, width = (sizes[name] for name in ("B", "S", "H", "Hkv", "N"))
    starts_at = {"q": 0, "k": heads * 64, "v": (heads + kv_heads) * 64}  # in packed
    elements = {"x": batch * seq * 256, "packed": batch * seq * width, "q_out": batch * heads * seq * 64,
                "k_out": batch * kv_heads * seq * 64, "context": batch * seq * heads * 64}

    def ends(tensor, counts, strides, row=64):
        last = starts_at.get(tensor, 0) + sum((n - 1) * stride for n, stride in zip(counts, strides)) + row
        packed_end = {"q": elements["packed"] - 2 * kv_heads * 64, "k": elements["packed"] - kv_heads * 64, "v": elements["packed"]}
        assert last == {**elements, **packed_end}[tensor], tensor

    linear = _example("sah_linear_w4", sizes)
    ends(linear["x"], [linear["rows"]], [linear["x_row_stride"]], linear["in_features"])
    ends(linear["y"], [linear["rows"]], [linear["y_row_stride"]], linear["out_features"])
    rotary = _example("sah_qk_norm_rotary", sizes)
    append = _example("sah_block_cache_append", sizes)
    attention = _example("sah_block_cache_attention", sizes)
    strides = lambda call, p: [call[f"{p}_stride_{axis}"] for axis in "bhs"]  # noqa: E731
    ends(rotary["query"], [batch, rotary["heads"], seq], strides(rotary, "q"))
    ends(rotary["key"], [batch, rotary["kv_heads"], seq], strides(rotary, "k"))
    ends(append["key"], [batch, append["kv_heads"], append["seq_len"]], strides(append, "k"))
    ends(append["value"], [batch, append["kv_heads"], append["seq_len"]], strides(append, "v"))
    ends(attention["query"], [batch, attention["heads"], attention["seq_len"]], strides(attention, "q"))
    ends(attention["output"], [batch, seq], [attention["o_stride_b"], attention["o_stride_s"]], heads * 64)


@pytest.mark.parametrize("shape", [(0, 128), (2, 0, 128), (0, 3, 128), (2, 0, 3, 128)])
def test_linear_w4_takes_no_rows(without_a_gpu, shape):
    check, arguments, _ = _requests()["linear"]
    assert check(**{**arguments, "value": torch.zeros(shape, dtype=torch.bfloat16)})

"""Plain 64-bit forms of the decoding operators, for their tests.

Written from the formulas, on CPU tensors of float64: the norm of a head with the
rotation, the block cache's coding, attention over what it stands for, and the
4-bit linear layer.  ``half_step`` is the largest relative error of one rounding.
"""

from __future__ import annotations

import math

import torch

BLOCK = 64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def norm_rotary(x, weight, bias, table, starts, *, norm, eps, interleaved):
    """x [B, H, S, D] in float64; table [positions, r] (cosines, sines) or None."""

    y = x.clone()
    if norm == "layer":
        y = y - y.mean(-1, keepdim=True)
    y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    if bias is not None:
        y = y + bias.double()
    if table is None:
        return y
    out = y.clone()
    half = table.shape[1] // 2
    for b in range(x.shape[0]):
        for s in range(x.shape[2]):
            position = (0 if starts is None else int(starts[b])) + s
            if not 0 <= position < table.shape[0]:
                out[b, :, s, : 2 * half] = math.nan
                continue
            cos, sin = table[position, :half].double(), table[position, half:].double()
            first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
            second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
            a, c = y[b, :, s, first], y[b, :, s, second]
            out[b, :, s, first] = a * cos - c * sin
            out[b, :, s, second] = c * cos + a * sin
    return out


def block_scale(block):
    """The scale of one block [64, D] of finite float64 values."""

    largest = float(block.abs().max())
    if largest == 0.0:
        return 1.0
    power = -100
    while largest / 2.0**power > 448.0:
        power += 1
    return 2.0**power


def e4m3(x):
    """Rounded to four significant bits, below 2^-6 to multiples of 2^-9, ties to even."""

    magnitude = x.abs().clamp(min=2.0**-6)
    step = torch.exp2(torch.floor(torch.log2(magnitude)) - 3)
    return torch.round(x / step) * step


def stored_tokens(key, value):
    """What the cache stands for after the tokens key, value [T, D] (float64) of one
    head: coded values in complete blocks, the tokens themselves behind them, and for
    a token that is not finite a key of NaN and a value of zeros."""

    bad = ~(torch.isfinite(key).all(-1) & torch.isfinite(value).all(-1))
    key, value = key.clone(), value.clone()
    key[bad] = 0.0
    value[bad] = 0.0
    for at in range(0, key.shape[0] // BLOCK * BLOCK, BLOCK):
        for x in (key, value):
            scale = block_scale(x[at : at + BLOCK])
            x[at : at + BLOCK] = e4m3(x[at : at + BLOCK] / scale) * scale
    key[bad] = math.nan
    return key, value


def attention(query, keys, values, position, scale):
    """One query row [D] over the tokens [T, D] up to ``position``: the answer, the
    same weights' sum of the values' magnitudes (what its errors are relative to),
    and 2^-36 of the largest weight on every value (a weight below 2^-25 of it is a
    subnormal fp16, in steps of 2^-24 / 2^11)."""

    scores = keys[: position + 1] @ query * scale
    weights = torch.softmax(scores, 0)
    sizes = values[: position + 1].abs()
    return weights @ values[: position + 1], (weights @ sizes, 2.0**-36 * weights.max() * sizes.sum(0))


def attention_bound(answer, sizes, query, keys, position, scale, dtype):
    """How far the kernel may be from ``answer``: the output's rounding; the weights'
    rounding to fp16 (relative 2^-11) and their relative error from the scores, twice
    that of a score: an fp32 sum of D products (D 2^-24 of their magnitudes) and one
    product by the scale; and 2^-20 for the fp32 sums over tokens and the exponential."""

    top = float((keys[: position + 1].abs() @ query.abs()).max()) * abs(scale)
    weights = 2.0**-11 + 2 * (query.shape[0] + 4) * 2.0**-24 * top + 2.0**-20
    inner = 2 * weights * sizes[0] + sizes[1]
    return half_step(dtype) * (answer.abs() + inner) + inner + 1e-30


def linear(x, weight, bias, gelu):
    """x [rows, K], weight [N, K] in float64; the answer and the magnitude of its terms."""

    out = x @ weight.t()
    magnitude = x.abs() @ weight.abs().t()
    if bias is not None:
        out, magnitude = out + bias, magnitude + bias.abs()
    if gelu:
        out = 0.5 * out * torch.erfc(-out / math.sqrt(2.0))
    return out, magnitude


def linear_bound(out, magnitude, inputs, gelu, dtype):
    """Output rounding and an fp32 sum of ``inputs`` products; GELU's slope is at most
    1.13 and its own error 1.7e-5 relative (with 1e-7 where it underflows)."""

    sums = (inputs + 16) * 2.0**-24 * magnitude
    if not gelu:
        return half_step(dtype) * (out.abs() + sums) + sums + 1e-30
    inner = 1.13 * sums + 1.7e-5 * out.abs() + 1e-7
    return half_step(dtype) * (out.abs() + inner) + inner

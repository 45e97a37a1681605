"""Verification of drafted tokens against the target's probabilities, on gfx950.

No counterpart in the reference, whose forward takes whole sequences.  A small model (or
a look-up) drafts a few tokens, the large one runs over them at once as a chunk
(solution/kernels/attention/hip_block_cache.py), and this operator says which of them stand
and what follows, so that the answer is distributed as the large model's own.
csrc/verify_draft.hip holds the kernels, include/shape_aware_hip.h the definition.

A step of one batch, behind ``starts`` tokens, with the token that the last step answered
and ``drafts`` drafted ones as its ``drafts + 1`` new tokens::

    answer, accepted, _ = hip_verify_draft(logits, tokens, uniforms, draft_logits)
    ends = starts + 1 + accepted          # what stays in the cache
"""

from __future__ import annotations

import torch

from ..hip._library import (
    HipLibraryError,
    differentiated,
    dtype_code,
    launch,
    library_available,
    library_for,
)

HIP_VERIFY_DRAFT_BACKEND = "hip_verify_draft"
SUPPORTED_DTYPES = frozenset({torch.float32, torch.float16, torch.bfloat16})
MAX_DRAFTS = 1024


def hip_verify_draft_available() -> bool:
    """Whether the gfx950 library loads in this process."""

    return library_available()


def _plain_ok(value: torch.Tensor | None, shape: tuple[int, ...], dtype: torch.dtype, index: int) -> bool:
    return value is None or (
        value.dtype is dtype and value.shape == shape and value.is_contiguous() and value.get_device() == index
    )


def _request(
    target: torch.Tensor,
    tokens: torch.Tensor,
    uniforms: torch.Tensor,
    draft: torch.Tensor | None,
    counts: torch.Tensor | None,
    temperatures: torch.Tensor | None,
) -> tuple | None:
    """The library, the device, the sizes and the workspace's bytes of a request that the
    kernels take, else None."""

    dtype, index, shape = target.dtype, target.get_device(), target.shape
    if dtype not in SUPPORTED_DTYPES or len(shape) != 3 or shape[1] < 1 or shape[2] < 1:
        return None
    batch, drafts, vocab = shape[0], shape[1] - 1, shape[2]
    if drafts > MAX_DRAFTS or (vocab > 1 and target.stride(2) != 1) or differentiated(target):
        return None
    if draft is not None and (
        draft.dtype is not dtype
        or draft.shape != (batch, drafts, vocab)
        or draft.get_device() != index
        or (vocab > 1 and draft.stride(2) != 1)
        or differentiated(draft)
    ):
        return None
    if tokens is None or uniforms is None or differentiated(uniforms):
        return None
    if temperatures is not None and differentiated(temperatures):
        return None
    if not (
        _plain_ok(tokens, (batch, drafts), torch.int64, index)
        and _plain_ok(uniforms, (batch, drafts + 1), torch.float32, index)
        and _plain_ok(counts, (batch,), torch.int32, index)
        and _plain_ok(temperatures, (batch,), torch.float32, index)
    ):
        return None
    library = library_for(index)
    if library is None:
        return None
    size = library.sah_verify_draft_workspace_bytes(batch, drafts, vocab, 0 if draft is None else 1)
    if batch and not size:  # more rows than a launch has workgroups for
        return None
    return library, index, batch, drafts, vocab, size


def can_use_hip_verify_draft(
    target: torch.Tensor,
    tokens: torch.Tensor,
    uniforms: torch.Tensor,
    draft: torch.Tensor | None = None,
    *,
    counts: torch.Tensor | None = None,
    temperatures: torch.Tensor | None = None,
) -> bool:
    """Whether the kernels take these tensors."""

    return _request(target, tokens, uniforms, draft, counts, temperatures) is not None


def hip_verify_draft(
    target: torch.Tensor,
    tokens: torch.Tensor,
    uniforms: torch.Tensor,
    draft: torch.Tensor | None = None,
    *,
    counts: torch.Tensor | None = None,
    temperatures: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, str]:
    """Which drafted tokens stand, and the token after them: ``(answer, accepted, marker)``.

    ``target`` [batch, drafts + 1, vocab] holds the answering model's logits, row i those
    after the first i drafted ``tokens`` [batch, drafts] (int64); ``draft`` [batch,
    drafts, vocab] the logits that these were drawn from, or None where the drafts are
    certain.  Both in bfloat16, float16 or float32 and of any strides, vocab contiguous.
    Draft i stands where those before it stand and ``uniforms[b, i] * q < p``, with its
    probabilities at ``temperatures`` [batch] (1 without; 0 takes the likeliest token).
    ``uniforms`` [batch, drafts + 1] (float32, in [0, 1)) draws the next token with its
    last number, from max(p - q, 0) behind a draft that does not stand, else from p.

    ``answer`` [batch, drafts + 1] (int64) holds the drafts that stand, the token drawn
    and -1 behind; ``accepted`` [batch] (int32) counts the former.  ``counts`` [batch]
    (int32) gives requests fewer drafts; below 0 a request takes no part (all -1).  A row
    with a logit of NaN or +inf, or none above -inf, answers -1 as the token drawn.  With
    no drafts (``tokens`` [batch, 0]) this draws one token a request.
    """

    request = _request(target, tokens, uniforms, draft, counts, temperatures)
    if request is None:
        raise RuntimeError("HIP draft verification is ineligible for the requested inputs")
    library, index, batch, drafts, vocab, size = request
    answer = tokens.new_empty((batch, drafts + 1))
    accepted = tokens.new_empty((batch,), dtype=torch.int32)
    try:
        workspace = tokens.new_empty(-(-size // 8)) if size else None
        launch(
            index,
            library.sah_verify_draft,
            "sah_verify_draft",
            target.data_ptr(),
            None if draft is None else draft.data_ptr(),
            tokens.data_ptr(),
            uniforms.data_ptr(),
            None if counts is None else counts.data_ptr(),
            None if temperatures is None else temperatures.data_ptr(),
            answer.data_ptr(),
            accepted.data_ptr(),
            batch,
            drafts,
            vocab,
            target.stride(0),
            target.stride(1),
            0 if draft is None else draft.stride(0),
            0 if draft is None else draft.stride(1),
            dtype_code(target.dtype),
            None if workspace is None else workspace.data_ptr(),
            size,
        )
    except HipLibraryError as exc:
        raise RuntimeError("HIP draft verification execution failed") from exc
    return answer, accepted, HIP_VERIFY_DRAFT_BACKEND


__all__ = [
    "HIP_VERIFY_DRAFT_BACKEND",
    "MAX_DRAFTS",
    "SUPPORTED_DTYPES",
    "can_use_hip_verify_draft",
    "hip_verify_draft",
    "hip_verify_draft_available",
]

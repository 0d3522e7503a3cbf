"""Scoring logits: log probabilities of given tokens, entropy, and the likeliest alternatives.

`token_logprobs` reads each row of logits once (ppyb200_token_logprobs): rows as the LM head writes
them (`GPT2.new_logits`, `GPT2.forward`, `GPT2.extend`), or any evenly spaced rows of f32, bf16 or
f16."""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import runtime
from .runtime import B200Error
from .torch_calls import begin, end

__all__ = ["TokenLogprobs", "token_logprobs"]

TOP_LIMIT = 64  # PPYB200_TOP_LIMIT


class TokenLogprobs(NamedTuple):
    """logprobs f32, shaped as the tokens; entropy f32 [...]; top_logprobs f32 and top_tokens int64
    [..., top], the largest first."""

    logprobs: object
    entropy: object
    top_logprobs: object
    top_tokens: object


#: Element types, as the header numbers them.
_KINDS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _rows(shape, strides) -> tuple[int, int]:
    """(rows, distance between rows) of [..., vocab] logits with evenly spaced rows; the distance is
    -1 where they are not."""
    if len(shape) == 2 and shape[0] > 1:
        return shape[0], strides[0]
    rows, pitch = 1, 0
    for size, stride in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if size != 1:
            if rows > 1 and stride != pitch * rows:
                return rows * size, -1
            pitch = stride if rows == 1 else pitch
        rows *= size
    return rows, pitch if rows > 1 else shape[-1]


def token_logprobs(logits, tokens, top: int = 0) -> TokenLogprobs:
    """Log probabilities of `tokens` under `logits` [..., vocab], each row's entropy (nats), and its
    `top` likeliest tokens (0 to 64) with their log probabilities.

    tokens int64 [...] (one a row) or [..., given] (several a row); a token outside the vocabulary
    (-1 where none is asked for) gives NaN. Alternatives come largest first, the lowest index
    first among equals, NaN above every number. A logit of -inf has probability 0; a row with a NaN
    or +inf, or with nothing above -inf, has NaN log probabilities and entropy."""
    kind, device = _KINDS.get(logits.dtype), logits.get_device()
    shape = logits.shape
    if kind is None or device < 0 or len(shape) < 1 or shape[-1] < 1:
        raise B200Error("logits: f32, bf16 or f16 [..., vocab] on a CUDA device")
    leading, vocab, strides = shape[:-1], shape[-1], logits.stride()
    rows, pitch = _rows(shape, strides)
    if pitch < vocab or (strides[-1] != 1 and vocab > 1):
        raise B200Error("logits: unit stride along the vocabulary, rows evenly spaced and at least "
                        "vocab elements apart")
    asked = tokens.shape
    several = len(asked) == len(shape)
    if (tokens.dtype is not torch.int64 or tokens.get_device() != device
            or not tokens.is_contiguous() or asked[:len(leading)] != leading
            or not (several or len(asked) == len(leading))):
        raise B200Error(f"tokens: contiguous int64 {list(leading)} or {list(leading)} + [given], "
                        f"on {logits.device}")
    if not 0 <= top <= min(TOP_LIMIT, vocab):
        raise B200Error(f"top: 0 up to {TOP_LIMIT} and the vocabulary")
    beside = begin(device)
    try:
        logprobs = torch.empty_like(tokens, dtype=torch.float32)
        result = TokenLogprobs(
            logprobs, logprobs.new_empty(leading) if several else torch.empty_like(logprobs),
            logprobs.new_empty((*leading, top)), tokens.new_empty((*leading, top)))
        if runtime.library().ppyb200_token_logprobs(
                logits.data_ptr(), kind, rows, vocab, pitch, tokens.data_ptr(),
                asked[-1] if several else 1, top, logprobs.data_ptr(), result[1].data_ptr(),
                result[2].data_ptr(), result[3].data_ptr()) != runtime.STATUS_OK:
            raise B200Error(runtime.last_error())
    finally:
        end(beside)
    return result

"""What a step's logits say of its tokens: log-probabilities of given tokens,
entropies and top alternatives.

The reference's engines read no more of the logits than their argmax
(hexgen2/model.py:79, 114); ``Engine.decode(on_logprobs=...)`` and
``Engine.score`` report these beside the tokens.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from . import _lib
from .fp4 import _call, _int32
from .ops import _DTYPES, _require_device


class TokenLogprobs(NamedTuple):
    """``logprob [...]`` of the given tokens (None without any), ``entropy
    [...]``, and ``top_logprobs`` / ``top_ids [..., top]`` of the likeliest
    tokens, likeliest first (None with ``top`` 0)."""
    logprob: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_logprobs: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


@functools.lru_cache(maxsize=1024)
def _form(shape, stride, dtype, top: int):
    """Rows, vocabulary, elements from row to row, type code and workspace bytes
    of a call."""
    if dtype not in _DTYPES or not shape or not shape[-1]:
        raise ValueError(f"logits must be [..., vocab] in float16, bfloat16 or float32, got {tuple(shape)} {dtype}")
    vocab = _int32(shape[-1], "vocab")
    if not 0 <= top <= min(_lib.MAX_TOP, vocab):
        raise ValueError(f"top {top} outside [0, {min(_lib.MAX_TOP, vocab)}]")
    if vocab > 1 and stride[-1] != 1:
        raise ValueError("logits rows must be contiguous")
    rows, step, span = shape.numel() // vocab, vocab, None
    for n, at in zip(reversed(shape[:-1]), reversed(stride[:-1])):
        if n == 1 or not rows:
            continue
        if span is None:
            step, span = at, at
        if at != span:
            raise ValueError("logits rows must lie at one stride")
        span *= n
    return rows, vocab, step, _DTYPES[dtype], int(_lib.load().hexkv_token_logprobs_workspace_bytes(rows, vocab, top))


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0) -> TokenLogprobs:
    """Score every row of ``logits [..., vocab]`` (float16, bfloat16 or
    float32; rows contiguous, at one stride) for ``tokens [...]`` (int64;
    a negative one is padding and scores 0, one past the vocabulary NaN): one pass
    over the logits, softmax sums in fp32, results float32 and int64.  A
    logit of -inf has probability 0; equal logits rank by lowest id."""
    _require_device(logits)
    top = int(top)
    rows, vocab, stride, dtype, need = _form(logits.shape, logits.stride(), logits.dtype, top)
    shape = logits.shape[:-1]
    if tokens is not None and (tokens.dtype != torch.int64 or tokens.shape != shape or tokens.device != logits.device
                               or not tokens.is_contiguous()):
        raise ValueError(f"tokens must be contiguous int64 {tuple(shape)} on {logits.device}")
    entropy = logits.new_empty(shape, dtype=torch.float32)
    logprob = None if tokens is None else torch.empty_like(entropy)
    values = ids = None
    if top:
        values = entropy.new_empty((*shape, top))
        ids = logits.new_empty((*shape, top), dtype=torch.int64)
    workspace = logits.new_empty(need, dtype=torch.uint8) if need else None
    _call("hexkv_token_logprobs", logits, logits.data_ptr(), stride, rows, vocab, dtype,
          None if tokens is None else tokens.data_ptr(), top, None if tokens is None else logprob.data_ptr(),
          entropy.data_ptr(), None if values is None else values.data_ptr(), None if ids is None else ids.data_ptr(),
          None if workspace is None else workspace.data_ptr(), need)
    return TokenLogprobs(logprob, entropy, values, ids)

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
from .fp4 import _call
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
def _workspace(rows: int, vocab: int, top: int) -> int:
    return int(_lib.load().hexkv_token_logprobs_workspace_bytes(rows, vocab, top))


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0) -> TokenLogprobs:
    """Score every row of ``logits [..., vocab]`` (float16, bfloat16 or
    float32; rows contiguous, at one stride) for ``tokens [...]`` (int64;
    a negative one is padding and scores 0, one past the vocabulary NaN): one pass
    over the logits, softmax sums in fp32, results float32 and int64.  A
    logit of -inf has probability 0; equal logits rank by lowest id."""
    _require_device(logits)
    if logits.dtype not in _DTYPES or logits.dim() < 1 or not logits.shape[-1]:
        raise ValueError(f"logits must be [..., vocab] in float16, bfloat16 or float32, got {tuple(logits.shape)} "
                         f"{logits.dtype}")
    shape, vocab, top = logits.shape[:-1], logits.shape[-1], int(top)
    if not 0 <= top <= min(_lib.MAX_TOP, vocab):
        raise ValueError(f"top {top} outside [0, {min(_lib.MAX_TOP, vocab)}]")
    if logits.is_contiguous() or logits.dim() == 1:
        stride = vocab
        if logits.dim() == 1 and vocab > 1 and logits.stride(0) != 1:
            raise ValueError("logits rows must be contiguous")
    elif logits.dim() == 2 and logits.stride(1) == 1:
        stride = logits.stride(0)
    else:
        raise ValueError("logits rows must be contiguous and lie at one stride")
    if tokens is not None and (tokens.dtype != torch.int64 or tokens.shape != shape or tokens.device != logits.device
                               or not tokens.is_contiguous()):
        raise ValueError(f"tokens must be contiguous int64 {tuple(shape)} on {logits.device}")
    rows = logits.numel() // vocab
    entropy = logits.new_empty(shape, dtype=torch.float32)
    logprob = None if tokens is None else torch.empty_like(entropy)
    values = ids = None
    if top:
        values = entropy.new_empty((*shape, top))
        ids = logits.new_empty((*shape, top), dtype=torch.int64)
    need = _workspace(rows, vocab, top)
    workspace = logits.new_empty(need, dtype=torch.uint8) if need else None
    _call("hexkv_token_logprobs", logits, logits.data_ptr(), stride, rows, vocab, _DTYPES[logits.dtype],
          None if tokens is None else tokens.data_ptr(), top, None if tokens is None else logprob.data_ptr(),
          entropy.data_ptr(), None if values is None else values.data_ptr(), None if ids is None else ids.data_ptr(),
          None if workspace is None else workspace.data_ptr(), need)
    return TokenLogprobs(logprob, entropy, values, ids)

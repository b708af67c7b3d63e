"""Rotary frequencies of a model's settings: what ``paged.append``, ``ops.rope_split``
and ``ops.norm_rope_linear`` turn q and k by.

The reference rotates by ``1 / base ** (2 j / dim)`` alone and refuses scaled
rotation (hexgen2/model.py:37-38); long-context models scale it.  ``paged.append``
takes the angle of a far position in 64 bits; ``ops.rope_split`` and
``ops.norm_rope_linear`` take position * frequency in fp32, off by up to 2^-24 of it.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

KINDS = ("default", "linear", "llama3", "yarn")


def kind_of(scaling: Optional[dict]) -> str:
    """Which of ``KINDS`` a model's ``rope_scaling`` names."""
    if not scaling:
        return "default"
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    if kind not in KINDS:
        raise ValueError(f"rotation scaled by {kind!r} is not supported (supported: {', '.join(KINDS)})")
    return kind


def _number(scaling: dict, name: str, default=None) -> float:
    value = scaling.get(name)
    if value is None:
        value = default
    if value is None or not float(value) > 0:
        raise ValueError(f"{scaling.get('rope_type', scaling.get('type'))} rotation needs a positive {name}, got {value!r}")
    return float(value)


def frequencies(dim: int, base: float = 10000.0, scaling: Optional[dict] = None,
                max_positions: Optional[int] = None, device=None) -> Tuple[torch.Tensor, float]:
    """``(inv_freq, scale)``: float32 ``[dim / 2]`` radians a position of the ``dim`` dims
    that turn, and what sines and cosines are multiplied by.

    ``scaling`` is a checkpoint's ``rope_scaling`` (``factor`` s throughout), for a
    frequency f = base ** (-2 j / dim), ``max_positions`` L0 the context it was
    trained for where ``scaling`` does not say (``original_max_position_embeddings``):

    * ``linear``: f / s;
    * ``llama3``: f where L0 f / 2 pi (its turns over L0) is above ``high_freq_factor``,
      f / s where it is below ``low_freq_factor``, between them mixed by where it lies;
    * ``yarn``: f where a pair makes more than ``beta_fast`` turns over L0, f / s below
      ``beta_slow``, between them mixed by the pair's place between those that make so many
      turns; scale ``attention_factor``, or 0.1 ln s + 1."""
    if dim < 0 or dim % 2 or not base > 0:
        raise ValueError(f"dim {dim} must be even and base {base} positive")
    kind = kind_of(scaling)
    # float32 powers of a float32 base, as checkpoints' own code has them
    f = 1.0 / (base ** (torch.arange(0, dim, 2, dtype=torch.float32) / dim)).double()
    scale = 1.0
    if kind == "linear":
        f = f / _number(scaling, "factor")
    elif kind == "llama3":
        s, length = _number(scaling, "factor"), _number(scaling, "original_max_position_embeddings", max_positions)
        low, high = _number(scaling, "low_freq_factor"), _number(scaling, "high_freq_factor")
        if not high > low:
            raise ValueError(f"llama3 rotation needs high_freq_factor {high} above low_freq_factor {low}")
        kept = ((length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = kept * f + (1 - kept) * f / s
    elif kind == "yarn":
        s, length = _number(scaling, "factor"), _number(scaling, "original_max_position_embeddings", max_positions)
        fast, slow = _number(scaling, "beta_fast", 32), _number(scaling, "beta_slow", 1)
        if any(scaling.get(k) is not None for k in ("mscale", "mscale_all_dim")) or scaling.get("truncate") is False:
            raise ValueError("yarn rotation with mscale, or with places that are not whole, is not supported")

        def pair(turns):  # the (fractional) pair that makes so many turns over L0
            return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))

        first, last = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
        kept = 1 - ((torch.arange(dim // 2, dtype=torch.float64) - first) / max(last - first, 0.001)).clamp(0, 1)
        f = kept * f + (1 - kept) * f / s
        scale = _number(scaling, "attention_factor", 0.1 * math.log(s) + 1 if s > 1 else 1.0)
    return f.float().to(device), scale

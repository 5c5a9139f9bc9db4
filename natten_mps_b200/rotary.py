"""Frequencies of rotary positions, for ``na1d_rotary`` and ``na1d_append``."""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, fast: float = 32.0, slow: float = 1.0,
                       device=None) -> Tuple[torch.Tensor, float]:
    """``(frequencies, magnitude)``: radians a position of the ``rotary_dim / 2`` channel pairs, ``base ** (-2 i /
    rotary_dim)`` in float64, and what the rotated channels are multiplied by (1 except for ``"yarn"``).

    ``scaling`` stretches them for contexts ``factor`` times as long as the ``original_length`` trained on:

    ``"linear"``  every frequency divided by ``factor`` (positions interpolated)
    ``"ntk"``     a larger base, ``base * factor ** (rotary_dim / (rotary_dim - 2))``: the slowest pair is divided by
                  ``factor``, the fastest kept
    ``"yarn"``    pairs that turn more than ``fast`` times within ``original_length`` kept, those that turn less than
                  ``slow`` times divided by ``factor``, a linear ramp over the pairs between; magnitude
                  ``0.1 ln(factor) + 1`` (Peng et al., "YaRN: Efficient context window extension of large language
                  models")
    """
    if isinstance(rotary_dim, bool) or not isinstance(rotary_dim, int) or rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even integer, got {rotary_dim}.")
    if not base > 1.0 or not math.isfinite(base):
        raise ValueError(f"base must be greater than 1, got {base}.")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}.")
    if not factor >= 1.0 or not math.isfinite(factor):
        raise ValueError(f"factor must be at least 1, got {factor}.")
    half, magnitude = rotary_dim // 2, 1.0
    if scaling == "ntk":
        if half < 2:
            raise ValueError("'ntk' scaling needs rotary_dim of at least 4.")
        base = base * factor ** (half / (half - 1))
    frequencies = [base ** (-i / half) for i in range(half)]
    if scaling == "linear":
        frequencies = [f / factor for f in frequencies]
    elif scaling == "yarn":
        if original_length is None or original_length < 1:
            raise ValueError("'yarn' scaling needs the original_length.")
        if not fast > slow > 0:
            raise ValueError("'yarn' scaling needs fast > slow > 0.")

        def pair(turns):                   # (fractional) index of the pair that turns so often within original_length
            return half * math.log(original_length / (turns * 2 * math.pi)) / math.log(base)

        low, high = max(0, math.floor(pair(fast))), min(rotary_dim - 1, math.ceil(pair(slow)))
        share = [min(1.0, max(0.0, (i - low) / max(high - low, 1e-3))) for i in range(half)]
        frequencies = [f * (1 - s) + f / factor * s for f, s in zip(frequencies, share)]
        magnitude = 0.1 * math.log(factor) + 1.0
    return torch.tensor(frequencies, dtype=torch.float64, device=device), magnitude


__all__ = ["rotary_frequencies"]

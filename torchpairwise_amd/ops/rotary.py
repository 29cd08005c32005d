"""Frequencies of rotary positions, as they are and stretched for longer contexts."""
from __future__ import annotations

import math

import torch

__all__ = ["rotary_frequencies"]

SCALINGS = ("none", "linear", "base", "parts")


def rotary_frequencies(width: int, base: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
                       original_length: int | None = None, fast: float = 32.0, slow: float = 1.0,
                       device=None) -> tuple[torch.Tensor, float]:
    """The float64 frequencies [width / 2] and the factor on the result that
    ``rotary_embedding(x, positions, frequencies, scale=...)`` takes.

    Pair ``i`` of ``width / 2`` turns by ``base ** (-2 i / width)`` a position.  ``scaling`` stretches
    them for contexts ``factor`` (>= 1) times as long as the ones they were made for:

    * ``"none"``: as they are (``factor`` must be 1);
    * ``"linear"``: every frequency divided by ``factor`` (positions interpolated);
    * ``"base"``: the base raised to ``base * factor ** (width / (width - 2))``, which leaves the
      fastest pair and divides the slowest one's frequency by ``factor``;
    * ``"parts"``: pairs that make ``fast`` turns or more over ``original_length`` positions stay, those
      that make ``slow`` or fewer are divided by ``factor``, with a linear ramp over the pairs between
      (from the last whole pair of the first to the first of the second, whether or not the width reaches
      them); the result is scaled by ``0.1 ln(factor) + 1``.
    """
    if width < 2 or width % 2:
        raise ValueError(f"rotary_frequencies: width must be even and at least 2, got {width}")
    if not (math.isfinite(base) and base > 1.0):
        raise ValueError(f"rotary_frequencies: base must be finite and above 1, got {base}")
    if scaling not in SCALINGS:
        raise ValueError(f"rotary_frequencies: scaling must be one of {SCALINGS}, got {scaling!r}")
    if not (math.isfinite(factor) and factor >= 1.0) or (scaling == "none" and factor != 1.0):
        raise ValueError(f"rotary_frequencies: factor {factor} does not fit scaling {scaling!r}")
    half = width // 2
    pair = torch.arange(half, dtype=torch.float64)
    scale = 1.0
    if scaling == "base" and width > 2:
        base = base * factor ** (width / (width - 2))
    frequencies = base ** (-pair / half)
    if scaling == "linear":
        frequencies = frequencies / factor
    elif scaling == "parts":
        if original_length is None or original_length < 1:
            raise ValueError("rotary_frequencies: scaling 'parts' needs original_length")
        if not fast > slow > 0:
            raise ValueError(f"rotary_frequencies: fast ({fast}) must be above slow ({slow}) and both positive")
        # the pair that makes t turns over the original length
        def pair_of(turns: float) -> float:
            return half * math.log(original_length / (2 * math.pi * turns)) / math.log(base)

        # not held to the pairs there are: an end moved inwards would change the slope
        first, last = math.floor(pair_of(fast)), math.ceil(pair_of(slow))
        ramp = ((pair - first) / max(last - first, 1)).clamp(0.0, 1.0)
        frequencies = frequencies * (1.0 - ramp) + frequencies / factor * ramp
        scale = 0.1 * math.log(factor) + 1.0
    return frequencies.to(device), scale

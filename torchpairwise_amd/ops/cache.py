"""The tensors of a cache of keys and values in 4 or 8 bits."""
from __future__ import annotations

import torch

__all__ = ["quantized_cache"]

BLOCK = 32  # features that share a scale
ROWS = 16  # rows come in multiples of this


def quantized_cache(batch: int, heads: int, rows: int, width: int, value_width: int | None = None, *, bits: int = 4,
                    device=None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Zeroed ``(key_codes, key_scales, value_codes, value_scales)`` that ``cache_write_``, ``cache_read`` and
    ``cache_attention`` take: room for ``rows`` rows of each of ``batch`` sequences, or ``batch`` pages of
    ``rows`` rows.  ``rows`` is a multiple of 16 (of pages: a power of two); ``width`` and ``value_width``
    (None: the same) are 1 to 256 features.

    Every 32 features of a row share a power of two 2^e, the first with which the largest magnitude is below
    7 * 2^e (``bits=4``) or 464 * 2^e (``bits=8``): halfway past the last code.  ``bits=4`` keeps values of 0, 0.5,
    1, 1.5, 2, 3, 4, 6 and a sign (uint8 codes, two a byte, the even feature in the low half), ``bits=8``
    float8_e4m3fn, rounded to nearest, ties to even; magnitudes that round to 2^128 (from 3.5 * 2^126 on, in 8 bits
    1.9375 * 2^127) read back as infinite, and attention makes infinities or NaN of them.  A feature takes
    ``bits + 0.25`` bits.
    Codes are ``[batch, heads, rows, bytes of whole blocks]``, scales (exponent + 127; 255: the block is NaN)
    ``[batch, heads, blocks, rows]``; any view of them with strides in multiples of 16 will do.
    """
    value_width = width if value_width is None else value_width
    if bits not in (4, 8):
        raise ValueError(f"quantized_cache: bits must be 4 or 8, got {bits}")
    if batch < 0 or heads < 1 or rows < 0 or rows % ROWS:
        raise ValueError(f"quantized_cache: batch must be at least 0, heads 1 and rows a multiple of {ROWS}, got "
                         f"{batch}, {heads} and {rows}")
    tensors = []
    for features in (width, value_width):
        if not 1 <= features <= 256:
            raise ValueError(f"quantized_cache: rows must have 1 to 256 features, got {features}")
        blocks = -(-features // BLOCK)
        codes = torch.zeros((batch, heads, rows, blocks * BLOCK * bits // 8), dtype=torch.uint8, device=device)
        tensors += [codes if bits == 4 else codes.view(torch.float8_e4m3fn),
                    torch.zeros((batch, heads, blocks, rows), dtype=torch.uint8, device=device)]
    return tuple(tensors)

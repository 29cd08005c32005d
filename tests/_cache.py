"""The cache in 4 or 8 bits from its definition, in 64 bits, and how far attention over it may be off.

What is stored is exact: a block's power of two and one rounding of x / 2^e have one right answer.

Attention: the values are exact in bfloat16, so the errors are those of tests/_attention.py, with more
terms where float32 queries and probabilities are three bfloat16 summands each (what three leave is below
2^-24 of the value):
  scores         |scale| (3 d + 4) u (|q_i| . |k_j|) + 4 u |s_ij|
  probabilities  relative: e_i = 2 max_j of that + (3 m + 16) u + b
  output         e_i (p |v|)_ij + b |o|
u = 2^-24, b the rounding of the data type.
"""
import math

import torch

from tests._attention import U, keep_of

BLOCK = 32
LAST = {4: 6.0, 8: 448.0}
PAST = {4: 7.0, 8: 464.0}  # values from here on round past the last code
FORMAT = {4: (1, 2, 1), 8: (3, 4, 7)}  # mantissa bits, exponent bits, bias


def two_to(e):
    return torch.ldexp(torch.ones((), dtype=torch.float64), e.double())


def blocks_of(width):
    return -(-width // BLOCK)


def stored(x, bits):
    """Rows [..., d] -> (exponents [..., blocks], values in units of the blocks' power [..., blocks, 32]) in
    64 bits; exponent 128 marks a block with NaN or an infinity."""
    d = x.shape[-1]
    x = torch.nn.functional.pad(x.double(), (0, -d % BLOCK)).unflatten(-1, (-1, BLOCK))
    bad = ~x.isfinite().all(-1)
    top = torch.where(bad, 0.0, x.abs().amax(-1))
    e = torch.frexp(top / PAST[bits])[1]
    e = torch.where(top == 0, -127, e.clamp(min=-127))
    y = torch.where(bad[..., None], 0.0, x / two_to(e)[..., None])
    mantissa, _, bias = FORMAT[bits]
    step = two_to((torch.frexp(y)[1] - 1).clamp(min=1 - bias) - mantissa)
    y = torch.round(y / step) * step
    assert (y.abs() <= LAST[bits]).all()
    return torch.where(bad, 128, e), y


def encode(x, bits):
    """Rows [..., d] -> bytes of the codes [..., whole blocks], scale bytes [..., blocks]."""
    e, y = stored(x, bits)
    mantissa, _, bias = FORMAT[bits]
    a = y.abs()
    ea = (torch.frexp(a)[1] - 1).clamp(min=1 - bias)
    fraction = a / two_to(ea)  # below 1: subnormal
    code = torch.where(fraction < 1, fraction * 2 ** mantissa, (fraction - 1) * 2 ** mantissa + (ea + bias) * 2 ** mantissa)
    code = code.long() + torch.signbit(y).long() * (8 if bits == 4 else 128)
    code = code.flatten(-2)
    if bits == 4:
        code = code[..., 0::2] + 16 * code[..., 1::2]
    return code.to(torch.uint8), (e + 127).to(torch.uint8)


def decode(codes, scales, bits, width):
    """Bytes [..., whole blocks] and scale bytes [..., blocks] -> 64-bit values [..., width]."""
    raw = codes.view(torch.uint8).long()
    if bits == 4:
        raw = torch.stack([raw % 16, raw // 16], -1).flatten(-2)
    mantissa, exponents, bias = FORMAT[bits]
    fraction, exponent = raw % 2 ** mantissa, raw // 2 ** mantissa % 2 ** exponents
    sign = 1.0 - 2.0 * (raw // 2 ** (mantissa + exponents)).double()
    y = sign * (fraction.double() / 2 ** mantissa + (exponent > 0)) * two_to(exponent.clamp(min=1) - bias)
    if bits == 8:
        y = torch.where(raw % 128 == 127, math.nan, y)
    s = torch.where(scales == 255, math.nan, two_to(scales.long() - 127))
    return (y.unflatten(-1, (-1, BLOCK)) * s[..., None]).flatten(-2)[..., :width]


def whole(codes, scales, bits, width, pages=None):
    """CPU tensors of a cache -> 64-bit [batch, heads, rows of a sequence, width] and which rows have a place
    [batch, rows]; zeros where they have none."""
    scales = scales.transpose(-1, -2)
    if pages is None:
        return decode(codes, scales, bits, width), torch.ones(codes.shape[0], codes.shape[2], dtype=torch.bool)
    there = (pages >= 0) & (pages < codes.shape[0])
    at = torch.where(there, pages, 0).long()
    c, s = codes.view(torch.uint8)[at], scales[at]  # [batch, pages, heads, rows, ...]
    y = decode(c, s, bits, width).masked_fill(~there[:, :, None, None, None], 0.0)
    return y.transpose(1, 2).flatten(2, 3), there.repeat_interleave(codes.shape[2], 1)


def reference(q, k, v, there, mask=None, causal=False, scale=None, lengths=None):
    """q [b, h, n, d], 64-bit k, v [b, heads, m, ...] (CPU) -> 64-bit output and its bound."""
    b_round = torch.finfo(q.dtype).eps / 2
    group, m, d = q.shape[1] // k.shape[1], k.shape[2], q.shape[3]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    keep = keep_of(q, k, mask, causal, lengths) & there[:, None, None, :]
    length = torch.full((q.shape[0],), m) if lengths is None else lengths.clamp(0, m)
    live = (torch.arange(m) < length[:, None]) & there
    k, v = (torch.where(live[:, None, :, None], x, 0.0).repeat_interleave(group, 1) for x in (k, v))
    q = q.double()
    s = scale * (q @ k.mT)
    if mask is not None and mask.dtype != torch.bool:
        s = s + mask.double()
    s = torch.where(keep, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = p @ v
    err_s = torch.where(keep, abs(scale) * (3 * d + 4) * U * (q.abs() @ k.abs().mT) + 4 * U * s.abs(), 0.0)
    e = 2 * err_s.amax(-1, keepdim=True) + (3 * m + 16) * U + b_round
    return o, e * (p @ v.abs()) + b_round * o.abs()

"""Plain 64-bit attention with its gradients, and how far a kernel's results may be from it.

The bounds are the rounding-error analysis of the formulas, element by element, u = 2^-24 and b the
rounding of the data type (half of its eps: 2^-8 for bfloat16, 2^-24 for float32):

  scores            ds_ij = |scale| (d + 2) u (|q_i| . |k_j|) + 4 u |s_ij|
  probabilities     relative: e_i = 2 max_j ds_ij + (m + 8) u + b (rounded for the matrix cores)
  output            e_i (p |v|)_ij + b |o|
  do . v, delta     (dv + 2) u |do| . |v|;  (dv + 2) u |do| . |o| + |do| . (the output's error)
  dscores           p (both errors) + |ds| (e_i + b)
  gradients         the dscores' (probabilities') error times |k|, |q| (|do|), sums of m (n * group)
                    terms in fp32, and b of the result
"""
import math

import torch

U = 2.0 ** -24


def keep_of(q, k, mask=None, causal=False, lengths=None):
    """bool [b, h, n, m]: pairs that are left (additive masks: all but -inf)."""
    b, h, n, m = q.shape[0], q.shape[1], q.shape[2], k.shape[2]
    keep = torch.ones(b, h, n, m, dtype=torch.bool)
    if mask is not None:
        keep = keep & (mask if mask.dtype == torch.bool else mask != -math.inf)
    length = torch.full((b,), m) if lengths is None else lengths.clamp(0, m)
    j, i = torch.arange(m), torch.arange(n)[:, None]
    keep = keep & (j < length.view(b, 1, 1, 1))
    if causal:
        keep = keep & (j - i <= (length - n).view(b, 1, 1, 1))
    return keep


def reference(q, k, v, mask=None, causal=False, scale=None, lengths=None, grad=None):
    """4-D operands on the CPU -> dict of the 64-bit results and their bounds (``tol_*``)."""
    b_round = torch.finfo(q.dtype).eps / 2
    group = q.shape[1] // k.shape[1]
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    keep = keep_of(q, k, mask, causal, lengths)
    m, n, d, dv = k.shape[2], q.shape[2], q.shape[3], v.shape[3]
    live = torch.arange(m) < (torch.full((q.shape[0],), m) if lengths is None else lengths.clamp(0, m)).view(-1, 1, 1)
    q, k, v = q.double(), k.double(), v.double()
    k, v = (torch.where(live[..., None], x, 0.0).repeat_interleave(group, 1) for x in (k, v))
    s = scale * (q @ k.mT)
    if mask is not None and mask.dtype != torch.bool:
        s = s + mask.double()
    s = torch.where(keep, s, -math.inf)
    top = s.amax(-1, keepdim=True) if m else s.new_full((*s.shape[:-1], 1), -math.inf)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    o = p @ v
    err_s = torch.where(keep, abs(scale) * (d + 2) * U * (q.abs() @ k.abs().mT) + 4 * U * s.abs(), 0.0)
    e = 2 * (err_s.amax(-1, keepdim=True) if m else 0.0) + (m + 8) * U + b_round
    tol_o = e * (p @ v.abs()) + b_round * o.abs()
    r = {"out": o, "tol_out": tol_o}
    if grad is None:
        return r
    g = grad.double()
    dp, delta = g @ v.mT, (g * o).sum(-1, keepdim=True)
    ds = torch.where(keep, p * (dp - delta), 0.0)
    err_dp = (dv + 2) * U * (g.abs() @ v.abs().mT)
    err_delta = (dv + 2) * U * (g.abs() * o.abs()).sum(-1, keepdim=True) + (g.abs() * tol_o).sum(-1, keepdim=True)
    err_ds = torch.where(keep, p * (err_dp + err_delta) + ds.abs() * (e + b_round), 0.0)

    def heads(x):  # sums over the query heads of a key head
        return x.unflatten(1, (-1, group)).sum(2)

    r["dq"] = scale * (ds @ k)
    r["tol_dq"] = abs(scale) * (err_ds @ k.abs() + m * U * (ds.abs() @ k.abs())) + b_round * r["dq"].abs()
    r["dk"] = scale * heads(ds.mT @ q)
    r["tol_dk"] = (abs(scale) * heads(err_ds.mT @ q.abs() + n * group * U * (ds.abs().mT @ q.abs())) +
                   b_round * r["dk"].abs())
    r["dv"] = heads(p.mT @ g)
    r["tol_dv"] = heads((p * e).mT @ g.abs() + n * group * U * (p.mT @ g.abs())) + b_round * r["dv"].abs()
    return r


def rotate(x, positions, frequencies, interleaved=False, scale=1.0, inverse=False):
    """64-bit rotary positions of x [b, h, n, d] (CPU)."""
    x, w = x.double(), 2 * frequencies.numel()
    t = positions.double().expand(x.shape[0], x.shape[2])[..., None] * frequencies.double()
    z = torch.polar(torch.full_like(t, scale), -t if inverse else t)[:, None]
    r = x[..., :w].unflatten(-1, (w // 2, 2) if interleaved else (2, w // 2))
    y = torch.complex(*r.unbind(-1 if interleaved else -2)) * z
    return torch.cat([torch.stack([y.real, y.imag], -1 if interleaved else -2).flatten(-2), x[..., w:]], -1)

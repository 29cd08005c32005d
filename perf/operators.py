"""Attention and rotary positions: the calls that these operators' speed is judged by.

A case is one pass through one operator, described by plain values.  ``run`` makes the calls of
this package where ``own`` is true and computes the same in elementary torch operations where it
is not.

Keys of a case
  op           "attention" or "rotary"
  dtype, grad  type of the data; grad: the forward and, for a given upstream gradient, its gradients
  b, h, n, d   sizes of the queries (of the rotated tensor): batch, heads, rows, width
  rows_first   the data lie as [b, n, h, d] and are given as transposed views
attention
  hk, m, dv    heads and rows of keys and values, width of the values (hk divides h)
  causal       the last query sees every key, the one before it all but the last, ...
  mask         "none", "keep" (boolean [n, m], some rows empty) or "bias" (added, fp32 [h, n, m])
  ragged       each batch entry has a length of its own between m / 2 and m
rotary
  width        features that are rotated, the others pass through
  interleaved  pairs of neighbours, or feature i with feature i + width / 2
  stretch      context extension factor (1: none)
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
BASE = 10000.0
ORIGINAL = 4096  # rows that the frequencies were made for before a context extension
KEEP = 0.25      # share of the pairs that a "keep" mask leaves


def _attention(dtype, grad, b, h, hk, n, m, d, dv=None, causal=False, mask="none", ragged=False,
               rows_first=False, name=None):
    case = {"op": "attention", "dtype": dtype, "grad": grad, "b": b, "h": h, "hk": hk, "n": n, "m": m, "d": d,
            "dv": d if dv is None else dv, "causal": causal, "mask": mask, "ragged": ragged,
            "rows_first": rows_first}
    return case if name is None else {"name": name, **case}


def _rotary(dtype, grad, b, h, n, d, width=None, interleaved=False, stretch=1.0, rows_first=False, name=None):
    case = {"op": "rotary", "dtype": dtype, "grad": grad, "b": b, "h": h, "n": n, "d": d,
            "width": d if width is None else width, "interleaved": interleaved, "stretch": stretch,
            "rows_first": rows_first}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # one new token of each of 16 sequences: launch and host time count
        _rotary("bf16", False, 16, 16, 1, 128, name="rotary_token"),
        # queries of a training batch, forward and gradient
        _rotary("bf16", True, 4, 16, 8192, 128, rows_first=True, name="rotary_train"),
        # odd sizes, part of the head, frequencies stretched for a longer context
        _rotary("fp32", True, 3, 5, 1003, 118, width=50, interleaved=True, stretch=4.0, name="rotary_odd"),
        # a few query vectors read a codebook of an odd size and width softly
        _attention("fp32", False, 1, 1, 1, 37, 1003, 50, name="attention_codebook"),
        # one new token of a few sequences over short caches: latency
        _attention("bf16", False, 4, 16, 4, 1, 1624, 128, ragged=True, name="attention_token"),
        # one new token of a serving batch over long caches: the memory's rate counts
        _attention("bf16", False, 16, 16, 2, 1, 32768, 128, ragged=True, rows_first=True,
                   name="attention_token_long"),
        # a chunk of new tokens over a cache, odd sizes
        _attention("bf16", False, 1, 16, 4, 500, 16384, 64, causal=True, name="attention_chunk"),
        # the batched configuration's sizes, every row against every row
        _attention("bf16", False, 1, 8, 8, 8192, 8192, 256, name="attention_batched"),
        # a training step's attention over a mini-batch of embeddings: launches count
        _attention("fp32", True, 1, 4, 4, 64, 64, 128, name="attention_minibatch_grad"),
        # a causal training step with shared key heads
        _attention("bf16", True, 2, 16, 4, 8192, 8192, 128, causal=True, rows_first=True,
                   name="attention_causal_grad"),
        # the batched configuration with gradients in full precision
        _attention("fp32", True, 1, 8, 8, 8192, 8192, 256, name="attention_batched_grad"),
        # attention over a neighbour graph of an odd number of points, isolated ones among them
        _attention("bf16", True, 1, 4, 4, 3001, 3001, 90, mask="keep", name="attention_neighbours_grad"),
    ]


def _size(rng, low, high):
    """A size between low and high, even over its logarithm; every other one a multiple of 32."""
    v = int(round(low * (high / low) ** rng.random()))
    return min(high, -(-v // 32) * 32) if rng.random() < 0.5 and high >= 32 else v


def draw(rng):
    dtype, rows_first = rng.choice(["bf16", "bf16", "fp32"]), rng.random() < 0.5
    b = rng.choice([1, 2, 3, 4, 8, 16])
    if rng.random() < 0.3:
        h, d, width = rng.choice([1, 2, 4, 8, 16, 5]), rng.choice([32, 50, 64, 96, 118, 128, 200, 256]), None
        if rng.random() < 0.4:
            width = 2 * rng.randint(1, d // 2)
        n = 1 if rng.random() < 0.25 else _size(rng, 2, 16384)
        while b * h * n * d > 4 * 16 * 8192 * 128:
            n = -(-n // 2)
        return _rotary(dtype, rng.random() < 0.5, b, h, n, d, width, rng.random() < 0.5,
                       rng.choice([1.0, 1.0, 2.0, 8.0]), rows_first)
    hk, group = rng.choice([1, 1, 2, 4, 8]), rng.choice([1, 1, 2, 4, 8])
    h, d = hk * group, rng.choice([32, 50, 64, 80, 90, 96, 128, 128, 192, 256])
    dv = d if rng.random() < 0.8 else rng.choice([16, 33, 64, 128])
    kind = rng.choice(["token", "chunk", "train", "train", "rows"])
    if kind == "token":  # one or a few new rows over a long cache
        n, m = rng.choice([1, 1, 2, 4]), _size(rng, 256, 65536)
        while b * hk * m * (d + dv) > 16 * 2 * 32768 * 256:
            m = -(-m // 2)
        return _attention(dtype, False, b, h, hk, n, m, d, dv, n > 1, "none", rng.random() < 0.7, rows_first)
    n, m, grad, ragged, causal, mask = _size(rng, 16, 8192), 0, kind == "train", False, False, "none"
    if kind == "chunk":
        m, causal, ragged = n + _size(rng, 1, 16384), True, rng.random() < 0.3
    elif kind == "train":
        m, causal, mask = n, rng.random() < 0.5, rng.choice(["none", "none", "keep", "bias"])
        ragged = mask == "none" and rng.random() < 0.3
    else:
        m, mask = _size(rng, 16, 8192), rng.choice(["none", "keep", "bias"])
    # no more products than the largest listed case, scores of at most 2^31 pairs
    while b * h * n * m * max(d, dv) > 8 * 8192 * 8192 * 256 or b * h * n * m > 1 << 31:
        if b > 1:
            b //= 2
        elif m == n:
            n = m = -(-n // 2)
        else:
            n, m = -(-n // 2), -(-m // 2)
    return _attention(dtype, grad, b, h, hk, n, max(m, n) if causal else m, d, dv, causal, mask, ragged, rows_first)


# ---------------------------------------------------------------- inputs
def _lengths(case):
    """Lengths between m / 2 and m, fixed by the sizes (a case's work does not change with the seed)."""
    rng = random.Random(case["m"] * 31 + case["b"])
    low = max(case["m"] // 2, case["n"] if case["causal"] else 1, 1)
    return [case["m"]] + [rng.randint(low, case["m"]) for _ in range(case["b"] - 1)]


def _rows(g, case, heads, rows, width):
    b, dtype = case["b"], DTYPES[case["dtype"]]
    if case["rows_first"]:
        return torch.randn(b, rows, heads, width, generator=g, device="cuda").to(dtype).transpose(1, 2)
    return torch.randn(b, heads, rows, width, generator=g, device="cuda").to(dtype)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, h, n, d = (case[k] for k in ("b", "h", "n", "d"))
    st = {"case": case}
    if case["op"] == "rotary":
        st["x"] = _rows(g, case, h, n, d)
        # each sequence stands somewhere in a context of its own
        start = torch.randint(0, int(ORIGINAL * case["stretch"]), (b, 1), generator=g, device="cuda")
        st["positions"] = start + torch.arange(n, device="cuda")
        st["gout"] = _rows(g, case, h, n, d) if case["grad"] else None
        return st
    st["q"] = _rows(g, case, h, n, d)
    st["k"], st["v"] = _rows(g, case, case["hk"], case["m"], d), _rows(g, case, case["hk"], case["m"], case["dv"])
    st["gout"] = _rows(g, case, h, n, case["dv"]) if case["grad"] else None
    st["mask"] = st["lengths"] = None
    if case["mask"] == "keep":  # every 16th row or so sees nothing
        m = torch.rand(n, case["m"], generator=g, device="cuda") < KEEP
        st["mask"] = m & (torch.rand(n, 1, generator=g, device="cuda") > 1 / 16)
    elif case["mask"] == "bias":  # a slope of its own over the distance for each head, and noise
        far = (torch.arange(n, device="cuda")[:, None] - torch.arange(case["m"], device="cuda")).abs().float()
        slope = 2.0 ** -torch.arange(1, h + 1, device="cuda").float()
        st["mask"] = torch.randn(h, n, case["m"], generator=g, device="cuda") - slope[:, None, None] * far
    if case["ragged"]:
        st["lengths"] = torch.tensor(_lengths(case), device="cuda")
    return st


def _frequencies(width, stretch):
    """Frequencies of the pairs: base^(-2 i / width) with the base raised so that the slowest pair
    turns `stretch` times as slowly; (frequencies in 64 bits, factor on the result)."""
    half = width // 2
    base = BASE * stretch ** (width / (width - 2)) if width > 2 else BASE
    factor = 1.0 if stretch == 1.0 else 0.1 * math.log(stretch) + 1.0
    return base ** (-torch.arange(half, dtype=torch.float64) / half), factor


def prepare(case, seed):
    st = _inputs(case, seed)
    if case["op"] == "rotary":
        st["frequencies"], st["factor"] = _frequencies(case["width"], case["stretch"])
        st["frequencies"] = st["frequencies"].cuda()
    if own and case["grad"]:
        for name in ("x", "q", "k", "v"):
            if name in st:
                st[name].requires_grad_()
    return st


# ---------------------------------------------------------------- plain forms
def _rotate(x, positions, frequencies, interleaved, factor):
    """x [b, h, n, d] in 32 bits; angles in the 64 bits of the frequencies, which a long context needs."""
    width = 2 * frequencies.numel()
    angle = (positions[..., None] * frequencies)[:, None]
    cos, sin = (angle.cos() * factor).float(), (angle.sin() * factor).float()
    r, rest = x[..., :width], x[..., width:]
    if interleaved:
        a, c = r[..., 0::2], r[..., 1::2]
        turned = torch.stack([a * cos - c * sin, a * sin + c * cos], dim=-1).flatten(-2)
    else:
        a, c = r[..., :width // 2], r[..., width // 2:]
        turned = torch.cat([a * cos - c * sin, a * sin + c * cos], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _plain_rotary(st):
    case = st["case"]
    y = _rotate(st["x"].float(), st["positions"], st["frequencies"], case["interleaved"], st["factor"])
    y = y.to(st["x"].dtype)
    if st["gout"] is None:
        return y
    back = _rotate(st["gout"].float(), -st["positions"], st["frequencies"], case["interleaved"], st["factor"])
    return y, back.to(st["x"].dtype)


def _keep(case, mask, lengths, device):
    """Pairs that are left, broadcast to [b, h, n, m], or None for all of them."""
    keep, n, m = None, case["n"], case["m"]
    if mask is not None and mask.dtype == torch.bool:
        keep = mask
    j = torch.arange(m, device=device)
    end = None if lengths is None else lengths[:, None, None, None]
    if end is not None:
        keep = (j < end) if keep is None else keep & (j < end)
    if case["causal"]:
        i = torch.arange(n, device=device)[:, None]
        seen = j - i <= (m if end is None else end) - n
        keep = seen if keep is None else keep & seen
    return keep


def _plain_attention(st):
    case, dtype = st["case"], st["q"].dtype
    b, h, hk, n, m, d, dv = (case[k] for k in ("b", "h", "hk", "n", "m", "d", "dv"))
    scale = 1.0 / math.sqrt(d)
    # the queries of the heads that share a key head are rows of one product
    q = st["q"].float().reshape(b, hk, h // hk * n, d)
    k, v = st["k"].float(), st["v"].float()
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).view(b, h, n, m)
    if case["mask"] == "bias":
        s += st["mask"]
    keep = _keep(case, st["mask"], st["lengths"], s.device)
    if keep is not None:
        s.masked_fill_(~keep, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.masked_fill_(total == 0, 1.0)).view(b, hk, -1, m)
    o = torch.matmul(p, v)
    out = o.view(b, h, n, dv).to(dtype)
    if st["gout"] is None:
        return out
    g = st["gout"].float().reshape(b, hk, h // hk * n, dv)
    gv = torch.matmul(p.transpose(-1, -2), g)
    gs = torch.matmul(g, v.transpose(-1, -2)).sub_((g * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    gq = torch.matmul(gs, k).view(b, h, n, d)
    gk = torch.matmul(gs.transpose(-1, -2), q)
    return out, gq.to(dtype), gk.to(dtype), gv.to(dtype)


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return _plain_rotary(state) if case["op"] == "rotary" else _plain_attention(state)
    import torchpairwise as tp

    if case["op"] == "rotary":
        x = state["x"]
        y = tp.rotary_embedding(x, state["positions"], state["frequencies"], interleaved=case["interleaved"],
                                scale=state["factor"])
        if state["gout"] is None:
            return y
        return y.detach(), *torch.autograd.grad(y, [x], state["gout"])
    q, k, v = state["q"], state["k"], state["v"]
    out = tp.attention(q, k, v, state["mask"], causal=case["causal"], lengths=state["lengths"])
    if state["gout"] is None:
        return out
    return out.detach(), *torch.autograd.grad(out, [q, k, v], state["gout"])


# ---------------------------------------------------------------- work
def _pairs(case):
    """Pairs of a query and a key that are left, over batch and heads."""
    n, m, pairs = case["n"], case["m"], 0
    for end in (_lengths(case) if case["ragged"] else [m] * case["b"]):
        if case["causal"]:  # row i of the n sees end - n + 1 + i keys
            first = max(0, n - end)
            pairs += sum((end - n + 1 + first, end)) * (n - first) // 2
        else:
            pairs += n * end
    return case["h"] * pairs * (KEEP * 15 / 16 if case["mask"] == "keep" else 1.0)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rotary":
        elements = case["b"] * case["h"] * case["n"] * case["d"]
        turned = case["b"] * case["h"] * case["n"] * case["width"]
        times = 2 if case["grad"] else 1
        return {"bytes": times * 2 * elements * size + case["b"] * case["n"] * 8, "flops": times * 3 * turned}
    b, h, hk, n, m, d, dv = (case[k] for k in ("b", "h", "hk", "n", "m", "d", "dv"))
    keys = sum(_lengths(case)) if case["ragged"] else b * m
    queries, rows = b * h * n * (d + dv), hk * keys * (d + dv)
    elements = queries + rows
    if case["grad"]:  # the upstream gradient in; the gradients out, zeros past a length too
        elements += b * h * n * (d + dv) + hk * b * m * (d + dv)
    mask = {"none": 0, "keep": n * m, "bias": 4 * h * n * m}[case["mask"]]
    pairs = _pairs(case)
    flops = 2 * pairs * (d + dv) + (2 * pairs * (3 * d + 2 * dv) if case["grad"] else 0)
    return {"bytes": elements * size + mask, "flops": int(flops)}


# ---------------------------------------------------------------- 64 bits
def _exact_rotary(case, st):
    freqs, factor = _frequencies(case["width"], case["stretch"])
    turns = st["positions"].double().unsqueeze(-1) * freqs.cuda()

    def turn(x, sign):
        z, w = x.double(), case["width"]
        r = z[..., :w]
        pairs = r.unflatten(-1, (w // 2, 2)) if case["interleaved"] else r.unflatten(-1, (2, w // 2)).transpose(-1, -2)
        c = torch.view_as_complex(pairs.contiguous())
        c = c * torch.polar(torch.full_like(turns, factor), sign * turns).unsqueeze(1)
        p = torch.view_as_real(c)
        p = p.flatten(-2) if case["interleaved"] else p.transpose(-1, -2).flatten(-2)
        return torch.cat([p, z[..., w:]], -1)

    y = turn(st["x"], 1.0)
    return y if st["gout"] is None else (y, turn(st["gout"], -1.0))


def _exact_attention(case, st):
    b, h, hk, n, m = (case[k] for k in ("b", "h", "hk", "n", "m"))
    q, k, v = (st[x].double() for x in ("q", "k", "v"))
    out = torch.zeros(b, h, n, case["dv"], dtype=torch.float64, device=q.device)
    grads = [torch.zeros_like(x) for x in (q, k, v)] if case["grad"] else []
    ends = _lengths(case) if case["ragged"] else [m] * b
    for bi in range(b):
        end = ends[bi]
        for hi in range(h):
            ki = hi // (h // hk)
            qq, kk, vv = (x.detach().clone().requires_grad_(case["grad"])
                          for x in (q[bi, hi], k[bi, ki, :end], v[bi, ki, :end]))
            logits = qq @ kk.mT / math.sqrt(case["d"])
            if case["mask"] == "bias":
                logits = logits + st["mask"][hi, :, :end].double()
            banned = torch.zeros(n, end, dtype=torch.bool, device=q.device)
            if case["mask"] == "keep":
                banned |= ~st["mask"][:, :end]
            if case["causal"]:
                banned |= torch.ones(n, end, dtype=torch.bool, device=q.device).triu(end - n + 1)
            empty = banned.all(-1, keepdim=True)
            logits = logits.masked_fill(banned & ~empty, -math.inf)
            o = torch.where(empty, 0.0, torch.softmax(logits, -1) @ vv)
            out[bi, hi] = o.detach()
            if case["grad"]:
                gq, gk, gv = torch.autograd.grad(o, [qq, kk, vv], st["gout"][bi, hi].double())
                grads[0][bi, hi] += gq
                grads[1][bi, ki, :end] += gk
                grads[2][bi, ki, :end] += gv
    return (out, *grads) if case["grad"] else out


def exact(case, seed):
    st = _inputs(case, seed)
    return _exact_rotary(case, st) if case["op"] == "rotary" else _exact_attention(case, st)

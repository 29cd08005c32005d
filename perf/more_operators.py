"""A cache of keys and values in 4 or 8 bits: the calls that its operators' speed is judged by.

A case is one pass through one operator, described by plain values.  ``run`` makes the calls of
this package where ``own`` is true and computes the same in elementary torch operations where it
is not.

The cache: every 32 features of a row share a power of two (a byte, its exponent + 127) and are held
as signed 4-bit values 0 .5 1 1.5 2 3 4 6 (two a byte, the even feature in the low half) or as
float8_e4m3fn.  codes [batch, heads, rows, whole blocks], scales [batch, heads, blocks, rows]; with
pages [pages, heads, rows of a page, ...] and a table [batch, pages of a sequence].

Keys of a case
  op           "store" (rows are written and read back), "read" (the whole cache) or "attend"
  dtype        type of the rows that are written, read back, asked with
  bits         4 or 8
  b, hk, m     sequences, heads of keys and values, rows that a sequence has room for
  d, dv        widths of the keys and the values
  page         rows of a page (0: the sequences' rows lie in one piece)
  ragged       lengths (of what is stored: counts) differ between the sequences
  rows_first   the data lie as [b, n, heads, d] and are given as transposed views
store, attend
  n            new rows a sequence (queries a sequence)
attend
  h            heads of the queries (a multiple of hk)
  causal       the last query sees every key, the one before it all but the last, ...
  mask         "none", "keep" (boolean [b, 1, 1, m]) or "bias" (added, fp32 [h, n, m])
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
BLOCK = 32
KEEP = 0.25  # share of the keys that a "keep" mask leaves


def _case(op, dtype, bits, b, hk, m, d, dv=None, page=0, ragged=False, rows_first=False, name=None, **more):
    case = {"op": op, "dtype": dtype, "bits": bits, "b": b, "hk": hk, "m": m, "d": d, "dv": d if dv is None else dv,
            "page": page, "ragged": ragged, "rows_first": rows_first, **more}
    return case if name is None else {"name": name, **case}


def _attend(dtype, bits, b, h, hk, n, m, d, dv=None, causal=False, mask="none", **more):
    return _case("attend", dtype, bits, b, hk, m, d, dv, h=h, n=n, causal=causal, mask=mask, **more)


def listed():
    return [
        # the new token of each of 16 sequences goes into a long cache: launch and host time count
        _case("store", "bf16", 4, 16, 2, 32768, 128, n=1, rows_first=True, name="store_token"),
        # the prompts of a batch, as the projections lay them out
        _case("store", "bf16", 4, 4, 16, 8192, 128, n=8192, rows_first=True, name="store_prompt"),
        # odd sizes, prompts of different lengths in a padded batch, pages
        _case("store", "fp32", 8, 3, 5, 2048, 118, dv=50, n=1003, page=64, ragged=True, name="store_odd"),
        # a whole cache read back, for a call that takes dense keys and values
        _case("read", "bf16", 4, 16, 2, 32768, 128, ragged=True, name="read_long"),
        # the same in 8 bits out of pages, few rows
        _case("read", "fp32", 8, 4, 4, 1664, 96, page=16, ragged=True, name="read_pages"),
        # one new token of a few sequences over short caches: latency
        _attend("bf16", 4, 4, 16, 4, 1, 1664, 128, ragged=True, name="attend_token"),
        # one new token of a serving batch over long caches: the memory's rate counts
        _attend("bf16", 4, 16, 16, 2, 1, 32768, 128, ragged=True, rows_first=True, name="attend_token_long"),
        # the same from 8 bits in pages
        _attend("bf16", 8, 16, 32, 8, 1, 8192, 128, page=64, ragged=True, name="attend_token_pages"),
        # full precision queries of an odd width that look up a quarter of the rows
        _attend("fp32", 4, 8, 16, 4, 1, 16000, 90, mask="keep", name="attend_lookup"),
        # a few drafted tokens a sequence, checked at once, an added value for every pair
        _attend("bf16", 4, 8, 16, 4, 4, 4096, 64, causal=True, mask="bias", name="attend_draft"),
        # a chunk of new tokens over a cache, odd sizes
        _attend("bf16", 4, 1, 16, 4, 500, 16384, 64, causal=True, name="attend_chunk"),
        # whole prompts over the cache that they have just filled
        _attend("bf16", 4, 2, 16, 4, 8192, 8192, 128, causal=True, rows_first=True, name="attend_prompt"),
    ]


def _size(rng, low, high, step=1):
    """A size between low and high, even over its logarithm, in whole steps."""
    v = int(round(low * (high / low) ** rng.random()))
    return min(high, -(-v // step) * step)


def draw(rng):
    op, dtype, bits = rng.choice(["store", "read", "attend", "attend", "attend"]), rng.choice(["bf16", "bf16", "fp32"]), rng.choice([4, 4, 8])
    b, hk, rows_first = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 2, 4, 5, 8]), rng.random() < 0.5
    d = rng.choice([32, 50, 64, 80, 90, 96, 118, 128, 128, 192, 256])
    dv = d if rng.random() < 0.8 else rng.choice([16, 33, 64, 128])
    page, ragged = rng.choice([0, 0, 16, 64, 256]), rng.random() < 0.6
    step = max(page, 16)
    m = _size(rng, 256, 65536, step)
    while b * hk * m * (d + dv) > 16 * 2 * 32768 * 256 * (1 if dtype == "bf16" else 0.5):
        m = -(-m // (2 * step)) * step
    if op == "read":
        return _case(op, dtype, bits, b, hk, m, d, dv, page, ragged, rows_first)
    if op == "store":
        n = 1 if rng.random() < 0.3 else _size(rng, 2, m)
        return _case(op, dtype, bits, b, hk, m, d, dv, page, ragged and n > 1, rows_first, n=n)
    h, mask = hk * rng.choice([1, 2, 4, 8, 16]), rng.choice(["none", "none", "none", "keep", "bias"])
    n = rng.choice([1, 1, 2, 4, _size(rng, 5, 8192)])
    # no more products than the largest listed case, scores of at most 2^31 pairs
    most = 2 * 16 * 4096 * 8192 * 128 // (1 if dtype == "bf16" else 8)
    while n > 1 and (n > m or b * h * n * m * max(d, dv) > most or b * h * n * m > 1 << 31):
        n = -(-n // 2)
    return _attend(dtype, bits, b, h, hk, n, m, d, dv, n > 1 and rng.random() < 0.7, mask, page=page, ragged=ragged,
                   rows_first=rows_first)


# ---------------------------------------------------------------- the cache in elementary operations
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _power(exponent):
    """2^(exponent - 127) in fp32 for whole numbers from 0 to 254, NaN for 255."""
    bits = torch.where(exponent == 0, 0x00400000, exponent << 23)
    return torch.where(exponent == 255, 0x7fc00000, bits).int().view(torch.float32)


def _quantised(x, bits):
    """Rows [..., n, d] -> codes [..., n, whole blocks], scales [..., n, blocks]."""
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))
    top = x.abs().amax(-1).view(torch.int32)
    # the first power of two that the largest value does not round past the last code with
    scale = ((top + 0x200000) >> 23) - 2 if bits == 4 else ((top + 0x180000) >> 23) - 8
    scale = torch.where(top >= 0x7f800000, 255, scale.clamp(min=0))
    y = x * _power(254 - scale.clamp(max=253))[..., None]
    y = torch.where((scale == 255)[..., None], 0.0, y).flatten(-2)
    if bits == 8:
        return y.to(torch.float8_e4m3fn), scale.to(torch.uint8)
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    code = torch.bucketize((a / step).round() * step, torch.tensor(MAGNITUDES, device=x.device))
    code = code.to(torch.uint8) + 8 * torch.signbit(y).to(torch.uint8)
    return code[..., 0::2] + 16 * code[..., 1::2], scale.to(torch.uint8)


def _values(codes, scales, bits, width):
    """Codes [..., n, whole blocks] and scales [..., n, blocks] -> fp32 [..., n, width]."""
    if bits == 8:
        x = codes.float()
    else:
        table = torch.tensor([*MAGNITUDES, *(-h for h in MAGNITUDES)], device=codes.device)
        x = table[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
    return (x.unflatten(-1, (-1, BLOCK)) * _power(scales.int())[..., None]).flatten(-2)[..., :width]


def _places(case, rows, pages):
    """First index and row of the cache's tensors for rows [b, n] of the sequences."""
    if not case["page"]:
        return torch.arange(case["b"], device=rows.device)[:, None].expand_as(rows), rows
    return pages.gather(1, rows // case["page"]).long(), rows % case["page"]


def _put(case, codes, scales, x, rows, live, pages):
    """Rows x [b, heads, n, d] to places `rows` [b, n], those of the indices `live` over [b * n] (None: all)."""
    c, s = _quantised(x, case["bits"])
    # float8 has no scatter of its own: bytes
    c, s = c.view(torch.uint8).transpose(1, 2).flatten(0, 1), s.transpose(1, 2).flatten(0, 1)
    first, row = (i.flatten() for i in _places(case, rows, pages))
    if live is not None:
        c, s, first, row = c[live], s[live], first[live], row[live]
    codes.view(torch.uint8).transpose(1, 2)[first, row] = c
    scales.permute(0, 3, 1, 2)[first, row] = s


def _get(case, codes, scales, width, rows, pages):
    """fp32 [b, heads, n, width] of places `rows` [b, n]."""
    first, row = _places(case, rows, pages)
    c = codes.view(torch.uint8).transpose(1, 2)[first, row].view(codes.dtype)
    return _values(c, scales.permute(0, 3, 1, 2)[first, row], case["bits"], width).transpose(1, 2)


def _whole(case, codes, scales, width, pages):
    """fp32 [b, heads, m, width] of everything."""
    if case["page"]:
        c, s = codes.view(torch.uint8)[pages.clamp(min=0)].view(codes.dtype), scales[pages.clamp(min=0)]
        c, s = c.transpose(1, 2).flatten(2, 3), s.permute(0, 2, 1, 4, 3).flatten(2, 3)
    else:
        c, s = codes, scales.transpose(-1, -2)
    return _values(c, s, case["bits"], width)


# ---------------------------------------------------------------- inputs
def _lengths(case):
    """Lengths between m / 2 and m, fixed by the sizes (a case's work does not change with the seed)."""
    if not case["ragged"]:
        return [case["m"]] * case["b"]
    rng = random.Random(case["m"] * 31 + case["b"])
    low = max(case["m"] // 2, case["n"] if case["op"] == "attend" and case["causal"] else 1, 1)
    return [case["m"]] + [rng.randint(low, case["m"]) for _ in range(case["b"] - 1)]


def _counts(case):
    """Rows of the padded batch that are stored, between n / 2 and n."""
    rng = random.Random(case["n"] * 31 + case["b"])
    return [rng.randint(max(case["n"] // 2, 1), case["n"]) if case["ragged"] else case["n"] for _ in range(case["b"])]


def _rows(g, case, heads, rows, width, dtype, spread=True):
    b = case["b"]
    shape = (b, rows, heads, width) if case["rows_first"] else (b, heads, rows, width)
    x = torch.randn(shape, generator=g, device="cuda")
    if spread:  # features of keys and values differ in size, as those of trained projections do
        by = torch.randn(heads, width, generator=g, device="cuda").mul_(0.5).exp_()
        x *= by if case["rows_first"] else by[:, None]
    x = x.to(dtype)
    return x.transpose(1, 2) if case["rows_first"] else x


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    b, hk, m, page = (case[k] for k in ("b", "hk", "m", "page"))
    dtype = DTYPES[case["dtype"]]
    st = {"case": case, "pages": None, "lengths": None, "mask": None}
    lengths = torch.tensor(_lengths(case), device="cuda")
    first, rows = (b, m) if not page else (b * (m // page), page)
    if page:
        st["pages"] = torch.randperm(first, generator=g, device="cuda").int().view(b, m // page)
        if case["op"] != "store":  # nothing stands in for pages past the end
            past = torch.arange(m // page, device="cuda") >= (lengths[:, None] + page - 1) // page
            st["pages"] = st["pages"].masked_fill(past, -1)
    st["cache"] = []
    for width in (case["d"], case["dv"]):
        blocks = -(-width // BLOCK)
        kind = torch.uint8 if case["bits"] == 4 else torch.float8_e4m3fn
        codes = torch.zeros(first, hk, rows, blocks * BLOCK * case["bits"] // 8, dtype=torch.uint8, device="cuda").view(kind)
        st["cache"] += [codes, torch.zeros(first, hk, blocks, rows, dtype=torch.uint8, device="cuda")]
    if case["op"] == "store":
        n = case["n"]
        st["key"], st["value"] = (_rows(g, case, hk, n, case[w], dtype) for w in ("d", "dv"))
        st["counts"] = torch.tensor(_counts(case), device="cuda") if case["ragged"] else None
        st["starts"] = torch.randint(0, m - n + 1, (b,), generator=g, device="cuda")
        return st
    # whole sequences, a few at a time (32 bits of all of them would be several times the cache)
    every = torch.arange(m, device="cuda").expand(1, m)
    for i in range(b):
        one = {**case, "b": 1, "rows_first": False}
        live = (every < lengths[i]).flatten().nonzero().flatten()
        pages = st["pages"][i:i + 1] if page else None
        for k, width in enumerate((case["d"], case["dv"])):
            codes, scales = st["cache"][2 * k:2 * k + 2]
            if not page:
                codes, scales = codes[i:i + 1], scales[i:i + 1]
            _put(one, codes, scales, _rows(g, one, hk, m, width, dtype), every, live, pages)
    if case["ragged"] or page:
        st["lengths"] = lengths
    if case["op"] == "attend":
        h, n = case["h"], case["n"]
        st["query"] = _rows(g, case, h, n, case["d"], dtype, spread=False)
        if case["mask"] == "keep":
            st["mask"] = torch.rand(b, 1, 1, m, generator=g, device="cuda") < KEEP
        elif case["mask"] == "bias":  # a slope of its own over distances up to 128 for each head, and noise
            far = (m - n + torch.arange(n, device="cuda")[:, None] - torch.arange(m, device="cuda")).abs().clamp(max=128).float()
            slope = 2.0 ** -torch.arange(1, h + 1, device="cuda").float()
            st["mask"] = torch.randn(h, n, m, generator=g, device="cuda") - slope[:, None, None] * far
    return st


def prepare(case, seed):
    return _inputs(case, seed)


# ---------------------------------------------------------------- plain forms
def _plain_store(st):
    case = st["case"]
    kc, ks, vc, vs = st["cache"]
    n, dtype = case["n"], st["key"].dtype
    i = torch.arange(n, device=kc.device)
    rows = st["starts"][:, None] + i
    live = None if st["counts"] is None else i < st["counts"][:, None]
    at = None if live is None else live.flatten().nonzero().flatten()
    got = []
    for codes, scales, x in ((kc, ks, st["key"]), (vc, vs, st["value"])):
        _put(case, codes, scales, x, rows, at, st["pages"])
        y = _get(case, codes, scales, x.shape[-1], rows, st["pages"])
        got.append((y if live is None else y * live[:, None, :, None]).to(dtype))
    return tuple(got)


def _plain_read(st):
    case = st["case"]
    kc, ks, vc, vs = st["cache"]
    got = []
    for codes, scales, width in ((kc, ks, case["d"]), (vc, vs, case["dv"])):
        y = _whole(case, codes, scales, width, st["pages"])
        if st["lengths"] is not None:
            off = torch.arange(case["m"], device=y.device) >= st["lengths"][:, None]
            y = y.masked_fill(off[:, None, :, None], 0.0)
        got.append(y.to(DTYPES[case["dtype"]]))
    return tuple(got)


def _plain_attend(st):
    case, dtype = st["case"], st["query"].dtype
    b, h, hk, n, m, d, dv = (case[k] for k in ("b", "h", "hk", "n", "m", "d", "dv"))
    kc, ks, vc, vs = st["cache"]
    k, v = _whole(case, kc, ks, d, st["pages"]), _whole(case, vc, vs, dv, st["pages"])
    # the queries of the heads that share a key head are rows of one product
    q = st["query"].float().reshape(b, hk, h // hk * n, d)
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).view(b, h, n, m)
    j = torch.arange(m, device=s.device)
    end = torch.full((b, 1, 1, 1), m, device=s.device) if st["lengths"] is None else st["lengths"][:, None, None, None]
    keep = j < end
    if case["causal"]:
        keep = keep & (j - torch.arange(n, device=s.device)[:, None] <= end - n)
    if case["mask"] == "keep":
        keep = keep & st["mask"]
    elif case["mask"] == "bias":
        s += st["mask"]
    s.masked_fill_(~keep, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.masked_fill_(total == 0, 1.0)).view(b, hk, -1, m)
    return torch.matmul(p, v).view(b, h, n, dv).to(dtype)


# ---------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return {"store": _plain_store, "read": _plain_read, "attend": _plain_attend}[case["op"]](state)
    import torchpairwise as tp

    cache, pages = state["cache"], state["pages"]
    widths = {"key_width": case["d"], "value_width": case["dv"], "dtype": DTYPES[case["dtype"]]}
    if case["op"] == "read":
        return tp.cache_read(*cache, **widths, counts=state["lengths"], pages=pages)
    if case["op"] == "attend":
        return tp.cache_attention(state["query"], *cache, state["mask"], causal=case["causal"],
                                  lengths=state["lengths"], pages=pages, value_width=case["dv"])
    starts, counts = state["starts"], state["counts"]
    tp.cache_write_(*cache, state["key"], state["value"], starts, counts=counts, pages=pages)
    return tp.cache_read(*cache, **widths, starts=starts, rows=case["n"], counts=counts, pages=pages)


# ---------------------------------------------------------------- work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    b, hk, m, d, dv = (case[k] for k in ("b", "hk", "m", "d", "dv"))
    held = sum(-(-w // BLOCK) * (BLOCK * case["bits"] // 8 + 1) for w in (d, dv))  # bytes of a row in the cache
    if case["op"] == "store":  # in, into the cache, out of it, out
        rows = hk * sum(_counts(case))
        return {"bytes": rows * (2 * held + (d + dv) * size) + hk * b * case["n"] * (d + dv) * size, "flops": 0}
    keys = sum(_lengths(case))
    if case["op"] == "read":
        return {"bytes": hk * (keys * held + b * m * (d + dv) * size), "flops": 0}
    h, n, pairs = case["h"], case["n"], 0
    for end in _lengths(case):
        if case["causal"]:  # row i of the n sees end - n + 1 + i keys
            first = max(0, n - end)
            pairs += (end - n + 1 + first + end) * (n - first) // 2
        else:
            pairs += n * end
    mask = {"none": 0, "keep": b * m, "bias": 4 * h * n * m}[case["mask"]]
    left = KEEP if case["mask"] == "keep" else 1.0
    return {"bytes": int(left * hk * keys * held) + b * h * n * (d + dv) * size + mask,
            "flops": int(2 * left * h * pairs * (d + dv))}


# ---------------------------------------------------------------- 64 bits
def _two_to(exponent):
    """2^exponent in 64 bits, exactly (a device's pow need not be)."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _exact_block_values(x, bits):
    """Rows [..., d] in 64 bits -> the values that the cache holds for them, from the definition: the
    block's step is the least power of two with which its largest value does not round past the last code."""
    last, past = (6.0, 7.0) if bits == 4 else (448.0, 464.0)  # last code; values from here on round past it
    mantissa, least = (1, 0) if bits == 4 else (3, -6)        # bits after the point; exponent of the smallest normal
    width = x.shape[-1]
    blocks = torch.nn.functional.pad(x.double(), (0, -width % BLOCK)).unflatten(-1, (-1, BLOCK))
    top = blocks.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(top / past)  # top / past in [2^(e-1), 2^e)
    e = torch.where(top == 0, -127, e.clamp(min=-127))
    y = blocks / _two_to(e)
    _, ey = torch.frexp(y)
    step = _two_to((ey - 1).clamp(min=least) - mantissa)
    y = (torch.round(y / step) * step).clamp(-last, last)
    return (y * _two_to(e)).flatten(-2)[..., :width]


def _exact_rows(codes, scales, bits, width):
    """One head's codes [n, bytes] and scales [n, blocks] -> 64-bit values [n, width], by the bits' meaning."""
    raw = codes.view(torch.uint8).long()
    if bits == 4:
        raw = torch.stack([raw % 16, raw // 16], -1).flatten(-2)
    mantissa, exponents, bias = (1, 2, 1) if bits == 4 else (3, 4, 7)
    fraction, exponent = raw % 2 ** mantissa, raw // 2 ** mantissa % 2 ** exponents
    sign = 1.0 - 2.0 * (raw // 2 ** (mantissa + exponents)).double()
    significand = fraction.double() / 2 ** mantissa + (exponent > 0)
    power = exponent.clamp(min=1) - bias + (scales.long() - 127).repeat_interleave(BLOCK, -1)
    return (sign * significand * _two_to(power))[:, :width]


def _exact_head(case, st, k, bi, hi):
    """Everything that sequence bi holds of head hi, [m, width]."""
    codes, scales = st["cache"][2 * k:2 * k + 2]
    width = case["dv"] if k else case["d"]
    if case["page"]:
        at = st["pages"][bi].clamp(min=0).long()
        c, s = codes.view(torch.uint8)[at, hi].flatten(0, 1), scales[at, hi].transpose(1, 2).flatten(0, 1)
    else:
        c, s = codes[bi, hi], scales[bi, hi].T
    return _exact_rows(c, s, case["bits"], width)


def exact(case, seed):
    st = _inputs(case, seed)
    b, hk, m = (case[k] for k in ("b", "hk", "m"))
    if case["op"] == "store":
        live = torch.arange(case["n"], device="cuda") < torch.tensor(_counts(case), device="cuda")[:, None]
        return tuple(_exact_block_values(st[x], case["bits"]) * live[:, None, :, None] for x in ("key", "value"))
    ends = _lengths(case)
    if case["op"] == "read":
        got = []
        for k, width in enumerate((case["d"], case["dv"])):
            y = torch.zeros(b, hk, m, width, dtype=torch.float64, device="cuda")
            for bi in range(b):
                for hi in range(hk):
                    y[bi, hi, :ends[bi]] = _exact_head(case, st, k, bi, hi)[:ends[bi]]
            got.append(y)
        return tuple(got)
    h, n = case["h"], case["n"]
    out = torch.zeros(b, h, n, case["dv"], dtype=torch.float64, device="cuda")
    for bi in range(b):
        end = ends[bi]
        banned = torch.zeros(n, end, dtype=torch.bool, device="cuda")
        if case["causal"]:
            banned |= torch.ones(n, end, dtype=torch.bool, device="cuda").triu(end - n + 1)
        if case["mask"] == "keep":
            banned |= ~st["mask"][bi, 0, :, :end]
        empty = banned.all(-1, keepdim=True)
        for ki in range(hk):
            kk, vv = (_exact_head(case, st, k, bi, ki)[:end] for k in (0, 1))
            for hi in range(ki * (h // hk), (ki + 1) * (h // hk)):
                logits = st["query"][bi, hi].double() @ kk.mT / math.sqrt(case["d"])
                if case["mask"] == "bias":
                    logits = logits + st["mask"][hi, :, :end].double()
                logits = logits.masked_fill(banned & ~empty, -math.inf)
                out[bi, hi] = torch.where(empty, 0.0, torch.softmax(logits, -1) @ vv)
    return out

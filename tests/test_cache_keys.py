"""cache_attention: every key counts once however the keys are split, float32 keeps all of its bits through the
summands of its products, and masks over pages of 16 rows."""
import math

import pytest
import torch

import torchpairwise as tp
from tests._attention import U
from tests._util import assert_close, gen
from tests.test_cache import attend, rows

F32, BF16 = torch.float32, torch.bfloat16
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


# ---------------------------------------------------------------- every key counts once
def chunk_counts(chunks, feature, width, limit):
    """64-bit means over keys 0 .. limit - 1 of values that are 1 at a key's chunk's feature and 0 elsewhere."""
    live = (limit - 32 * torch.arange(chunks)).clamp(0, 32).double()
    return torch.zeros(width, dtype=torch.float64).index_add_(0, feature, live) / max(limit, 1)


SHAPES = [(1, 240), (1, 4096), (1, 40912), (4, 8208), (12, 24704), (20, 24704), (40, 24704), (300, 8208)]  # rows, keys


@pytest.mark.parametrize("device,n,m", [("cpu", *x) for x in SHAPES[:4]] +
                         [pytest.param("cuda", *x, marks=pytest.mark.gpu) for x in SHAPES])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits,d", [(4, 64), (4, 128), (8, 128), (4, 256)])
def test_every_chunk_of_keys_counts_once(device, dtype, bits, d, n, m):
    """A query of zeros weighs every key alike, and the values of 32 keys are 1 at one feature: a feature of the
    output says how often the chunks that share it were counted.  Two assignments of features: chunks that share one
    in the first share none in the second (the second's run is a stretch of neighbours).

    Scores of 0 make weights of exactly 1, sums of at most 40912 ones are exact in 32 bits, the quotient is off by
    its division, its product and the type's rounding: 4 u and half a step of the type."""
    chunks, b_round = -(-m // 32), torch.finfo(dtype).eps / 2
    query = torch.zeros(1, 2, n, d, dtype=dtype, device=device)
    lengths = torch.tensor([m - 7], device=device)
    starts = torch.zeros(1, dtype=torch.long, device=device)
    each = -(-chunks // d)
    for feature in (torch.arange(chunks) % d, torch.arange(chunks) // each):
        value = torch.nn.functional.one_hot(feature.repeat_interleave(32)[:m], d).to(BF16).view(1, 1, m, d).to(device)
        cache = tp.quantized_cache(1, 1, m, d, bits=bits, device=device)
        tp.cache_write_(*cache, torch.ones_like(value), value, starts)
        for causal in (False, True):
            out = tp.cache_attention(query, *cache, causal=causal, lengths=lengths).cpu().double()
            limits = [m - 7 - (n - 1 - i if causal else 0) for i in range(n)]
            want = torch.stack([chunk_counts(chunks, feature, d, x) for x in limits])
            tol = want * (4 * U + b_round)
            # a chunk less or more: 32 / m of the output's sum of 1
            assert 32.0 / m > 4 * tol.max()
            assert_close(out, want.expand(1, 2, n, d), rtol=0.0, atol=tol.expand(1, 2, n, d), what=f"{causal}")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("page", [16, 32, 256])
@pytest.mark.parametrize("n", [1, 12, 100])
def test_every_chunk_in_pages_counts_once(dtype, page, n):
    """The same over a batch of ragged lengths in pages, some of which are not there."""
    b, m, d, b_round = 4, 8192, 128, torch.finfo(dtype).eps / 2
    per, chunks = m // page, m // 32
    pages = torch.randperm(b * per, generator=gen(3)).view(b, per)
    lengths = torch.tensor([m, 5003, 33, 2048])
    feature = torch.arange(chunks) % d
    value = torch.nn.functional.one_hot(feature.repeat_interleave(32), d).to(BF16).expand(b, 1, m, d).cuda()
    cache = tp.quantized_cache(b * per, 1, page, d, device="cuda")
    tp.cache_write_(*cache, torch.ones_like(value), value, torch.zeros(b, dtype=torch.long, device="cuda"), pages=pages.cuda())
    gone = torch.rand(b, per, generator=gen(4)) < 0.2
    pages[gone] = -1
    out = tp.cache_attention(torch.zeros(b, 2, n, d, dtype=dtype, device="cuda"), *cache, lengths=lengths.cuda(),
                             pages=pages.cuda())
    keep = (torch.arange(m) < lengths[:, None]) & ~gone.repeat_interleave(page, 1)
    want = torch.stack([torch.zeros(d, dtype=torch.float64).index_add_(0, feature.repeat_interleave(32), k.double()) /
                        k.sum().clamp_min(1) for k in keep])[:, None, None].expand(b, 2, n, d)
    assert_close(out, want, rtol=0.0, atol=want * (4 * U + b_round))


# ---------------------------------------------------------------- float32 keeps its bits
ROWS = [1, 3, 4, 5, 16, 17, 32, 33, 64, 65, 200]  # of a key head: one kernel each for 4, 16, 32, 64 (wide rows), more


def two_keys(bits, d, dv, key, device):
    """A cache whose keys 0 and 1 are zeros and `key` in every feature ([b] of them), with values 0 and 1."""
    b = len(key)
    k, v = torch.zeros(b, 1, 16, d), torch.zeros(b, 1, 16, dv)
    k[:, 0, 1] = torch.tensor(key)[:, None]
    v[:, 0, 1] = 1.0
    cache = tp.quantized_cache(b, 1, 16, d, dv, bits=bits, device=device)
    tp.cache_write_(*cache, k.to(device), v.to(device), torch.zeros(b, dtype=torch.long, device=device))
    assert (tp.cache_read(*cache, key_width=d, value_width=dv, dtype=F32)[0].cpu() == k).all()
    return cache


def share(s):
    """exp(s) / (1 + exp(s)) and how far float32 may be off: the exponent's product with log2 e by 3 u of itself, its
    power by 2 u, the sum by 2 u, the division by 2 u and the last product by u."""
    o = torch.sigmoid(s)
    return o, o * (3 * s.abs() + 12) * U


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("n", ROWS)
def test_every_bit_of_a_float32_query_counts(device, bits, d, n):
    """Queries of 1 + 3 2^-e and -1 against keys of 2^e: a score of 3 that the query's bits from 2^-e on decide, those
    of its first, second or third summand of 8 bits.  Every product and sum is a whole number below 2^25 and exact."""
    ends = (7, 15, 23)
    cache = two_keys(bits, d, d, [2.0 ** e for e in ends], device)
    q = torch.zeros(3, 1, n, d)
    at = torch.randint(0, d, (n,), generator=gen(n))
    for b, e in enumerate(ends):
        q[b, 0, torch.arange(n), at] = 1 + 3 * 2.0 ** -e
        q[b, 0, torch.arange(n), (at + 1 + torch.arange(n) % (d - 1)) % d] = -1.0
    out = tp.cache_attention(q.to(device), *cache, scale=1.0, lengths=torch.full((3,), 2, device=device))
    o, tol = share(torch.full((3, 1, n, d), 3.0, dtype=torch.float64))
    assert (o - 0.5).min() > 8 * tol.max()  # of a score of 0, without them
    assert_close(out, o, rtol=0.0, atol=tol)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("n", ROWS)
def test_every_bit_of_a_float32_probability_counts(device, bits, d, n):
    """Scores of 0 and -t: the second key's weight exp(-t) alone reaches the output, with all of its bits."""
    cache = two_keys(bits, d, d, [1.0], device)
    t = torch.rand(1, 8, n, generator=gen(n + 50))
    q = torch.zeros(1, 8, n, d)
    q.scatter_(3, torch.randint(0, d, (1, 8, n, 1), generator=gen(n)), -t[..., None])
    # 8 heads one by one: as many rows a key head as n
    out = torch.cat([tp.cache_attention(q[:, h:h + 1].to(device), *cache, scale=1.0, lengths=torch.tensor([2], device=device))
                     for h in range(8)], 1)
    o, tol = (x[..., None].expand(1, 8, n, d) for x in share(-t.double()))
    # two summands of 8 bits would be seen
    p = torch.exp(-t.double()).float()
    cut = (p.view(torch.int32) & ~0xff).view(F32).double() / (1 + p.double())
    assert ((cut - o[..., 0]).abs() > 4 * tol[..., 0]).any()
    assert_close(out, o, rtol=0.0, atol=tol)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("n", [x for x in ROWS if x <= 16])
def test_few_bfloat16_rows_are_rounded_once(device, bits, d, n):
    """The same of bfloat16: probabilities are off by 2^-17 (two summands), and the output is rounded, half a step."""
    cache = two_keys(bits, d, d, [1.0], device)
    t = torch.rand(1, 32, n, generator=gen(n + 70)).to(BF16)
    q = torch.zeros(1, 32, n, d, dtype=BF16)
    q.scatter_(3, torch.randint(0, d, (1, 32, n, 1), generator=gen(n)), -t[..., None])
    out = torch.cat([tp.cache_attention(q[:, h:h + 1].to(device), *cache, scale=1.0, lengths=torch.tensor([2], device=device))
                     for h in range(32)], 1)
    o, tol = (x[..., None].expand(1, 32, n, d) for x in share(-t.double()))
    tol = tol + 2.0 ** -17 * o + torch.ldexp(torch.ones_like(o), torch.frexp(o)[1] - 9)  # half a step of o's binade
    # one summand would be seen: rounded twice
    p = torch.exp(-t.double())
    once = (p.to(BF16).double() / (1 + p)).to(BF16).double()[..., None]
    assert n < 3 or ((once - o[..., :1]).abs() > tol[..., :1]).any()
    assert_close(out, o, rtol=0.0, atol=tol)


# ---------------------------------------------------------------- masks, over pages of 16 rows too
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [50, 128, 224])
@pytest.mark.parametrize("n", [1, 3, 8, 10, 16, 40])
@pytest.mark.parametrize("paged", [True, False])
def test_masks_by_widths_and_pages(dtype, bits, d, n, paged):
    """Two heads a key head, short caches and long ones, a sequence with holes, lengths that end inside a page; and
    the same rows in one piece."""
    b, h, hk = 2, 4, 2
    for m in (48, 240, 1104):
        first, pages, g = b, None, gen(m + n)
        if paged:
            first = b * (m // 16) + 1
            pages = torch.randperm(first, generator=gen(m))[:b * (m // 16)].view(b, -1).int()
            pages[1, ::3] = -1
            pages[1, 1] = first
        keep = torch.rand(b, h, n, m, generator=g) < 0.5
        keep[0, 0, 0] = False
        bias = torch.randn(b, h, n, m, generator=g)
        bias[torch.rand(b, h, n, m, generator=g) < 0.3] = -math.inf
        for what, mask in (("keep", keep), ("keys", keep[:, :1, :1]), ("bias", bias), ("bf16", bias[:, :, :1].to(BF16))):
            for causal in (False, True):
                attend("cuda", rows(b, h, n, d, 1, dtype), first, hk, m, d, bits, mask, causal,
                       lengths=torch.tensor([m - 5, m]), pages=pages, spoil=True, what=f"{m} {what} {causal}")


# ---------------------------------------------------------------- the borders of the scale
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits,border", [(4, 7.0), (8, 464.0)])
def test_the_power_that_a_border_takes(device, dtype, bits, border):
    """The first power 2^e with which the largest magnitude is below the border."""
    below = torch.tensor(border, dtype=dtype)
    below = (below * (1 - torch.finfo(dtype).eps / 2)).float().item()
    assert below < border
    x = torch.zeros(1, 1, 16, 32, dtype=dtype)
    for i, (top, e) in enumerate(((border, -3), (border, 0), (border, 60), (below, -3), (below, 0), (below, 60))):
        x[0, 0, i, i] = -top * 2.0 ** e
        x[0, 0, i, 31] = 2.0 ** (e - 9)  # the smallest of 8 bits with the smaller power, half of it with the larger
    cache = tp.quantized_cache(1, 1, 16, 32, bits=bits, device=device)
    tp.cache_write_(*cache, x.to(device), x.to(device), torch.zeros(1, dtype=torch.long, device=device))
    assert cache[1][0, 0, 0, :6].tolist() == [125, 128, 188, 124, 127, 187]
    got = tp.cache_read(*cache, dtype=F32)[0].cpu()[0, 0, :, 31]
    assert got[:3].eq(0).all()
    assert (got[3:6] == (torch.tensor([2.0 ** -12, 2.0 ** -9, 2.0 ** 51]) if bits == 8 else 0.0)).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits,first", [(4, 3.5 * 2.0 ** 126), (8, 1.9375 * 2.0 ** 127)])
def test_magnitudes_that_round_past_float32(device, dtype, bits, first):
    """From `first` on finite magnitudes round to 2^128; the one before stays finite."""
    before = torch.tensor(first * (1 - torch.finfo(dtype).eps / 2), dtype=torch.float64).to(dtype)
    assert before.double() < first
    x = torch.zeros(1, 1, 16, 32, dtype=dtype)
    x[0, 0, 0, 0], x[0, 0, 1, 0], x[0, 0, 2, 0] = first, -torch.finfo(dtype).max, before
    cache = tp.quantized_cache(1, 1, 16, 32, bits=bits, device=device)
    tp.cache_write_(*cache, x.to(device), x.to(device), torch.zeros(1, dtype=torch.long, device=device))
    for y in (*tp.cache_read(*cache, dtype=F32), *tp.cache_read(*cache)):
        assert y[0, 0, 0, 0] == math.inf and y[0, 0, 1, 0] == -math.inf and y[0, 0, 2, 0].isfinite()
        assert (y[..., 1:] == 0).all()

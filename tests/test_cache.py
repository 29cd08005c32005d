"""cache_write_, cache_read and cache_attention: what is stored bit for bit, attention within the bounds of
tests/_cache.py, layouts, pages, what is left alone, and refusals."""
import ctypes as C
import math

import pytest
import torch
from torch.autograd import forward_ad

import torchpairwise as tp
from torchpairwise_amd import _capi as capi
from tests import _cache as ref
from tests._util import assert_close, assert_equal, gen

F32, BF16, F8 = torch.float32, torch.bfloat16, torch.float8_e4m3fn
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TINY = 1e-30
PATTERN = 0x55


def like(x, device):
    """A copy on the device with the same strides."""
    if x is None:
        return None
    y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=device)
    y.copy_(x)
    return y


def rows(b, h, n, d, seed, dtype=F32, rows_first=False):
    """Rows whose features differ in size."""
    x = torch.randn((b, n, h, d) if rows_first else (b, h, n, d), generator=gen(seed))
    x = (x * torch.randn(d, generator=gen(seed + 100)).mul(0.5).exp()).to(dtype)
    return x.transpose(1, 2) if rows_first else x


def empty_cache(first, heads, n, d, dv, bits, device, rows_first=False):
    """Cache tensors filled with a pattern; rows_first: rows before heads in memory."""
    out = []
    for w in (d, dv):
        blocks = ref.blocks_of(w)
        shape = (first, n, heads, blocks * 4 * bits) if rows_first else (first, heads, n, blocks * 4 * bits)
        codes = torch.full(shape, PATTERN, dtype=torch.uint8, device=device)
        codes = codes.transpose(1, 2) if rows_first else codes
        out += [codes if bits == 4 else codes.view(F8),
                torch.full((first, heads, blocks, n), PATTERN, dtype=torch.uint8, device=device)]
    return out


def raw(x):
    return x.view(torch.uint8).cpu()


def filled(first, heads, n, d, dv, bits, device, seed=5, rows_first=False):
    """A cache of random rows that the oracle has encoded: (CPU tensors, device tensors)."""
    cpu = empty_cache(first, heads, n, d, dv, bits, "cpu", rows_first)
    for k, w in enumerate((d, dv)):
        codes, scales = ref.encode(rows(first, heads, n, w, seed + k), bits)
        cpu[2 * k].view(torch.uint8).copy_(codes)
        cpu[2 * k + 1].copy_(scales.transpose(-1, -2))
    return cpu, [like(x.view(torch.uint8), device).view(x.dtype) for x in cpu]


# ---------------------------------------------------------------- what is stored
def edge_rows(bits, dtype):
    """Blocks at the borders of the format: [1, 1, n, 64]."""
    past, last = ref.PAST[bits], ref.LAST[bits]
    g = gen(11)
    grid = torch.arange(0, 33) / 4.0 if bits == 4 else torch.arange(0, 33) / 1.0
    blocks = []
    for e in (-149, -135, -130, -127, -126, -125, -30, 0, 3, 100, 119, 124, 125):
        unit = math.ldexp(1.0, e)
        for lead in (last, past, past * (1 - 2.0 ** -23), past * (1 + 2.0 ** -23), past * (1 - 2.0 ** -7), last / 2):
            x = torch.randn(32, generator=g, dtype=torch.float64) * last / 4
            x[:16] = grid[1:17] * (1 if bits == 4 else 13) * (1 - 2 * (torch.arange(16) % 2))  # ties among them
            x[20] = lead
            blocks.append(x.clamp(-lead, lead) * unit)
    for special in (0.0, -0.0, 1e-45, 2.0 ** -126, 3.4028234663852886e38, -3.4028234663852886e38, math.nan, -math.nan,
                    math.inf, -math.inf):
        x = torch.zeros(32, dtype=torch.float64)
        x[7] = special
        blocks.append(x)
        blocks.append(x + torch.randn(32, generator=g, dtype=torch.float64) * (torch.arange(32) != 7))
    if len(blocks) % 2:
        blocks.append(torch.zeros(32, dtype=torch.float64))
    return torch.stack(blocks).view(1, 1, -1, 64).to(F32).to(dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_stored_at_the_borders_of_the_format(device, bits, dtype):
    x = edge_rows(bits, dtype)
    n = x.shape[2]
    cache = empty_cache(1, 1, -(-n // 16) * 16, 64, 64, bits, device)
    tp.cache_write_(*cache, x.to(device), -x.to(device), torch.zeros(1, dtype=torch.long, device=device))
    for k, y in enumerate((x, -x)):
        codes, scales = ref.encode(y, bits)
        assert_equal(raw(cache[2 * k])[:, :, :n], codes, "codes")
        assert_equal(raw(cache[2 * k + 1])[..., :n], scales.transpose(-1, -2), "scales")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_every_code_and_scale_is_read(device, bits, dtype):
    """All 256 bytes of codes under all 256 scales."""
    bytes_ = 4 * bits
    codes = torch.arange(256, dtype=torch.uint8).view(1, 256 // bytes_, 1, bytes_).expand(1, -1, 256, -1).contiguous()
    scales = torch.arange(256, dtype=torch.uint8).view(1, 1, 1, 256).expand(1, 256 // bytes_, 1, 256).contiguous()
    want = ref.decode(codes, scales.transpose(-1, -2), bits, 32).float().to(dtype)
    c = codes.to(device)
    c = c if bits == 4 else c.view(F8)
    got = tp.cache_read(c, scales.to(device), c, scales.to(device), dtype=dtype)
    for y in got:
        assert y.dtype == dtype
        assert_equal(y, want, nan_payload=False)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [4, 8])
def test_values_are_off_by_half_a_step_at_most(device, bits):
    x = rows(2, 3, 50, 100, 3)
    cache = tp.quantized_cache(2, 3, 64, 100, bits=bits, device=device)
    tp.cache_write_(*cache, x.to(device), x.to(device), torch.tensor([0, 14], device=device))
    for y in tp.cache_read(*cache, key_width=100, value_width=100, dtype=F32, rows=50,
                           starts=torch.tensor([0, 14], device=device)):
        e, _ = ref.stored(x, bits)
        mantissa, _, bias = ref.FORMAT[bits]
        # of the value's binade, or of the block's smallest one
        least = ref.two_to(e + 1 - bias - mantissa).repeat_interleave(32, -1)[..., :100] / 2
        half = torch.maximum(2.0 ** -(mantissa + 1) * x.double().abs(), least)
        assert ((y.cpu().double() - x.double()).abs() <= half).all()


# ---------------------------------------------------------------- where it goes
WRITES = [  # b, heads, rows, n, d, dv, bits, rows first (new rows), rows first (cache)
    (3, 2, 32, 1, 128, 128, 4, True, False),
    (2, 3, 48, 17, 64, 64, 4, False, True),
    (1, 1, 16, 16, 33, 200, 4, False, False),
    (2, 2, 64, 37, 118, 50, 8, True, True),
    (1, 4, 32, 5, 256, 32, 8, False, False),
    (2, 1, 80, 70, 1, 97, 4, True, False),
    (2, 2, 32, 31, 192, 160, 8, True, False),
]


def places(starts, counts, n, capacity, pages, first, page):
    """{(sequence, i): (entry, row)} of the rows that have a place."""
    out = {}
    for b, s in enumerate(starts):
        for i in range(min(n, counts[b]) if counts is not None else n):
            j = s + i
            if not 0 <= j < capacity:
                continue
            at = (b, j) if pages is None else (int(pages[b][j // page]), j % page)
            if 0 <= at[0] < first:
                out[b, i] = at
    return out


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", WRITES, ids=str)
@pytest.mark.parametrize("paged", [False, True])
def test_rows_go_to_their_places_and_nowhere_else(device, dtype, size, paged):
    """Starts before, inside and behind the cache, counts, pages that are not there; every other byte stays."""
    b, h, m, n, d, dv, bits, rf, cf = size
    page, first, pages = m, b, None
    if paged:
        page, per, first = 16, m // 16, b * (m // 16) + 2
        pages = torch.randperm(first, generator=gen(4))[:b * per].view(b, per)
        pages[0, 0] = -1
        pages[-1, -1] = first
        pages = pages.int() if bits == 4 else pages
    key, value = rows(b, h, n, d, 1, dtype, rf), rows(b, h, n, dv, 2, dtype, rf)
    cache = empty_cache(first, h, page if paged else m, d, dv, bits, device, cf)
    starts = [3, -2, m - 1][:b] if b > 1 else [0]
    counts = [max(n - 2, 0), n, n + 5][:b]
    at = places(starts, counts, n, m, pages, first, page)
    want = [raw(x).clone() for x in cache]
    for k, x in enumerate((key, value)):
        codes, scales = ref.encode(x, bits)
        for (bi, i), (f, r) in at.items():
            want[2 * k][f, :, r] = codes[bi, :, i]
            want[2 * k + 1][f, :, :, r] = scales[bi, :, i]
    args = dict(counts=torch.tensor(counts, device=device), pages=None if pages is None else pages.to(device))
    s = torch.tensor(starts, device=device)
    assert tp.cache_write_(*cache, like(key, device), like(value, device), s, **args) is None
    for x, w in zip(cache, want):
        assert_equal(raw(x), w)
    # and out again
    got = tp.cache_read(*cache, key_width=d, value_width=dv, dtype=dtype, starts=s, rows=n, **args)
    for k, (y, width) in enumerate(zip(got, (d, dv))):
        expected = torch.zeros(b, h, n, width, dtype=dtype)
        for (bi, i), (f, r) in at.items():
            expected[bi, :, i] = ref.decode(want[2 * k][f, :, r], want[2 * k + 1][f, :, :, r], bits, width).to(dtype)
        assert y.dtype == dtype
        assert_equal(y, expected)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_of_any_layout_are_written(device):
    """Rows that start at odd addresses, lie apart, or whose features do."""
    b, h, n, d = 2, 3, 9, 64
    base = torch.randn(b, h, n, 2 * d + 3, generator=gen(1))
    for x in (base[..., 1:d + 1], base[..., 3:d + 3], base[..., :2 * d:2], base[:, :, :1].expand(b, h, n, 2 * d + 3)[..., :d],
              base.transpose(2, 3)[:, :, :n, :n].repeat(1, 1, 1, 8)[..., :d], base[:1].expand(b, h, n, 2 * d + 3)[..., 2:d + 2]):
        for dtype in (F32, BF16):
            y = x.to(dtype) if x.to(dtype) is x else like(x.to(dtype), "cpu")
            cache = tp.quantized_cache(b, h, 16, d, device=device)
            on = base.to(device)  # the view itself where the type is the same
            z = torch.as_strided(on, x.shape, x.stride(), x.storage_offset()) if dtype == F32 and \
                x.untyped_storage().data_ptr() == base.untyped_storage().data_ptr() else y.to(device)
            tp.cache_write_(*cache, z, z, torch.zeros(b, dtype=torch.int32, device=device))
            codes, scales = ref.encode(x.to(dtype), 4)
            for k in (0, 1):
                assert_equal(raw(cache[2 * k])[:, :, :n], codes)
                assert_equal(raw(cache[2 * k + 1])[..., :n], scales.transpose(-1, -2))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [3, 70, 1000])
@pytest.mark.parametrize("widths", [(32, 256), (256, 32), (96, 160)], ids=str)
def test_keys_and_values_of_very_different_widths(device, n, widths):
    """The narrower rows need fewer blocks than the wider ones: those behind the last row do nothing."""
    x = [rows(3, 2, n, w, 60 + k, BF16) for k, w in enumerate(widths)]
    cache = empty_cache(3, 2, 1008, *widths, 4, device)
    s = torch.full((3,), 5, device=device)
    tp.cache_write_(*cache, *(y.to(device) for y in x), s)
    got = tp.cache_read(*cache, key_width=widths[0], value_width=widths[1], starts=s, rows=n)
    for k in (0, 1):
        codes, scales = ref.encode(x[k], 4)
        want, want_scales = (torch.full(y.shape, PATTERN, dtype=torch.uint8) for y in cache[2 * k:2 * k + 2])
        want[:, :, 5:5 + n], want_scales[..., 5:5 + n] = codes, scales.transpose(-1, -2)
        assert_equal(raw(cache[2 * k]), want)
        assert_equal(raw(cache[2 * k + 1]), want_scales)
        assert_equal(got[k], ref.decode(codes, scales, 4, widths[k]).to(BF16))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [1, 70])
def test_starts_and_counts_at_the_ends_of_their_type(device, n):
    least, most = -2 ** 63, 2 ** 63 - 1
    starts = torch.tensor([least, least + 1, most, most - 1, 0, 0, 0], device=device)
    counts = torch.tensor([most, most, most, most, least, least + 1, most], device=device)
    x = rows(7, 2, n, 64, 70)
    cache = empty_cache(7, 2, 80, 64, 64, 8, device)
    before = [raw(y).clone() for y in cache]
    tp.cache_write_(*cache, x.to(device), x.to(device), starts, counts=counts)
    codes, scales = ref.encode(x[6:], 8)
    for k, (y, w) in enumerate(zip(cache, before)):
        if k % 2:
            w[6:, :, :, :n] = scales.transpose(-1, -2)
        else:
            w[6:, :, :n] = codes
        assert_equal(raw(y), w)
    for y in tp.cache_read(*cache, dtype=F32, starts=starts, rows=n, counts=counts):
        assert (y[:6] == 0).all() and (y[6] != 0).any()


@pytest.mark.parametrize("device", DEVICES)
def test_a_page_shared_by_sequences_is_read_by_both(device):
    cpu, cache = filled(4, 2, 16, 64, 64, 4, device)
    pages = torch.tensor([[2, 0], [2, 3]], dtype=torch.int32)
    k, v = tp.cache_read(*cache, dtype=F32, pages=pages.to(device))
    want, _ = ref.whole(cpu[0], cpu[1], 4, 64, pages)
    assert_equal(k, want.float())
    q = rows(2, 2, 1, 64, 9)
    wv, there = ref.whole(cpu[2], cpu[3], 4, 64, pages)
    o, tol = ref.reference(q, want, wv, there)
    assert_close(tp.cache_attention(q.to(device), *cache, pages=pages.to(device)), o, rtol=0.0, atol=tol + TINY)


# ---------------------------------------------------------------- attention
def attend(device, q, first, hk, m, dv, bits, mask=None, causal=False, scale=None, lengths=None, pages=None,
           rows_first=False, spoil=False, seed=5, what=""):
    """cache_attention against the oracle; spoil: rows past the lengths hold whatever is worst."""
    b, d = q.shape[0], q.shape[3]
    page = m if pages is None else m // pages.shape[1]
    cpu, cache = filled(first, hk, page, d, dv, bits, device, seed, rows_first)
    k, there = ref.whole(cpu[0], cpu[1], bits, d, pages)
    v, _ = ref.whole(cpu[2], cpu[3], bits, dv, pages)
    if spoil:
        for bi in range(b):
            length = m if lengths is None else int(lengths[bi].clamp(0, m))
            for j in range(length, m):
                f, r = (bi, j) if pages is None else (int(pages[bi][j // page]), j % page)
                if 0 <= f < first:
                    for side in (0, 2):
                        cache[side].view(torch.uint8)[f, :, r] = 0x7f
                        cache[side + 1][f, :, :, r] = 255
    o, tol = ref.reference(q, k, v, there, mask, causal, scale, lengths)
    dev = lambda x: None if x is None else x.to(device)  # noqa: E731
    out = tp.cache_attention(like(q, device), *cache, dev(mask), causal=causal, scale=scale, lengths=dev(lengths),
                             pages=dev(pages), value_width=dv)
    assert out.dtype == q.dtype and out.shape == (*q.shape[:3], dv)
    assert_close(out, o, rtol=0.0, atol=tol + TINY, what=what)
    return out


SIZES = [  # b, heads, key heads, n, m, d, dv, rows first
    (1, 1, 1, 1, 16, 1, 1, False),
    (2, 4, 4, 1, 64, 128, 128, True),
    (3, 8, 1, 1, 1008, 64, 64, False),
    (1, 16, 2, 3, 336, 128, 96, True),      # 24 rows a key head
    (2, 16, 1, 1, 128, 50, 50, False),      # 16 rows
    (1, 4, 2, 16, 144, 33, 200, False),     # 32 rows
    (2, 2, 1, 5, 80, 256, 256, True),
    (1, 32, 2, 1, 96, 192, 160, False),
    (1, 4, 2, 33, 160, 64, 64, True),       # 66 rows: tiles
    (2, 3, 3, 70, 272, 128, 128, False),
    (1, 4, 1, 50, 208, 90, 33, True),
    (1, 2, 2, 130, 144, 256, 256, False),
    (1, 6, 2, 40, 400, 160, 192, False),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_attention(device, dtype, bits, causal, size):
    b, h, hk, n, m, d, dv, rf = size
    attend(device, rows(b, h, n, d, 1, dtype, rf), b, hk, m, dv, bits, causal=causal, rows_first=rf)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [1, 4, 20])
@pytest.mark.parametrize("paged", [0, 16, 64])
def test_lengths_and_what_lies_behind_them(device, dtype, bits, n, paged):
    """Lengths of 0 and 1, past m and below 0, ends inside a page and inside eight keys; rows behind them are
    NaN and are not read."""
    b, h, hk, m, d = 7, 4, 2, 320, 64
    lengths = torch.tensor([0, 1, 31, 256, 317, 999, -5])
    pages = None
    if paged:
        pages = torch.randperm(b * m // paged, generator=gen(2)).view(b, m // paged)
    out = attend(device, rows(b, h, n, d, 1, dtype), b if not paged else b * m // paged, hk, m, d, bits, lengths=lengths,
                 pages=pages, causal=n > 1, spoil=True)
    assert not out[0].any() and not out[6].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("mask", [None, "keep", "bias"])
def test_pages_that_are_not_there_hold_no_keys(device, dtype, bits, n, mask):
    b, h, hk, m, d, page = 3, 4, 2, 256, 96, 32
    pages = torch.randperm(30, generator=gen(3))[:b * 8].view(b, 8).int()
    pages[0, 2] = -1
    pages[0, 7] = 30
    pages[1] = -7  # nothing at all
    pages[2, 0] = 2 ** 31 - 1
    if mask == "keep":
        mask = torch.rand(b, 1, n, m, generator=gen(4)) < 0.4
    elif mask == "bias":
        mask = torch.randn(h, n, m, generator=gen(4))
    out = attend(device, rows(b, h, n, d, 1, dtype), 30, hk, m, d, bits, mask, pages=pages,
                 lengths=torch.tensor([250, 256, 130]))
    assert not out[1].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kind", ["none", "keep", "bias"])
@pytest.mark.parametrize("n,page", [(9, 0), (16, 16), (17, 0), (30, 64), (32, 0), (33, 0)])
def test_wide_float32_rows_in_groups(device, bits, kind, n, page):
    """More than 128 features of float32: 16 rows a block up to 64, then tiles."""
    b, h, hk, m, d, dv = 2, 4, 2, 320, 200, 136
    mask = None
    if kind != "none":
        mask = torch.randn(b, h, n, m, generator=gen(7))
        mask = mask > -0.3 if kind == "keep" else mask
    pages, first = None, b
    if page:
        first = b * (m // page) + 1
        pages = torch.randperm(first, generator=gen(8))[:b * (m // page)].view(b, -1).int()
    attend(device, rows(b, h, n, d, 90), first, hk, m, dv, bits, mask, causal=kind == "none",
           lengths=torch.tensor([m - 3, 70]), pages=pages, spoil=True)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 90, 128, 256])
@pytest.mark.parametrize("n", [1, 9, 45])
@pytest.mark.parametrize("kind", ["keep", "keep_keys", "bias", "bias_heads", "bias_bf16", "strided"])
def test_masks(device, dtype, d, n, kind):
    b, h, hk, m = 2, 4, 2, 112
    g = gen(7)
    if kind == "keep":
        mask = torch.rand(n, m, generator=g) < 0.4
        mask[n // 2] = False  # a row that nothing is left to
        mask[-1] = torch.arange(m) == 17  # one key
    elif kind == "keep_keys":
        mask = torch.rand(b, 1, 1, m, generator=g) < 0.5
        mask[1] = False
    elif kind == "strided":
        mask = (torch.rand(b, h, m, n, generator=g) < 0.5).mT
    elif kind == "bias":
        mask = torch.randn(n, m, generator=g)
        mask[torch.rand(n, m, generator=g) < 0.3] = -math.inf
        if n > 1:
            mask[1] = -math.inf
            mask[2] = torch.finfo(F32).min  # the lowest value: every key weighs the same
            mask[3, 1:] = torch.finfo(F32).min
    elif kind == "bias_heads":
        mask = torch.randn(h, 1, 1, generator=g) * 3 + torch.zeros(1)
    else:
        mask = torch.randn(1, h, n, m + 1, generator=g).to(BF16)[..., 1:]
    attend(device, rows(b, h, n, d, 1, dtype), b, hk, m, d, 4, mask, what=kind)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("additive", [False, True])
def test_keys_that_a_mask_leaves_out_may_be_nan(device, bits, n, additive):
    """NaN and infinite keys, their values finite, behind a mask."""
    b, h, m, d = 1, 2, 80, 64
    q = rows(b, h, n, d, 1)
    cpu, cache = filled(b, h, m, d, d, bits, device)
    k, there = ref.whole(cpu[0], cpu[1], bits, d)
    v, _ = ref.whole(cpu[2], cpu[3], bits, d)
    off = torch.zeros(m, dtype=torch.bool)
    off[[0, 33, 79]] = True
    mask = torch.where(off, -math.inf, 0.0).expand(n, m) if additive else ~off.expand(n, m)
    o, tol = ref.reference(q, k, v, there, mask)
    cache[1][0, :, 0, off.to(device)] = 255
    assert_close(tp.cache_attention(q.to(device), *cache, mask.to(device)), o, rtol=0.0, atol=tol)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [1, 40])
def test_nan_spreads_to_the_rows_that_see_it(device, n):
    q = rows(1, 2, n, 64, 1)
    cpu, cache = filled(1, 2, 64, 64, 64, 4, device)
    cache[1][0, 1, 0, 5] = 255  # a key of the second head
    out = tp.cache_attention(q.to(device), *cache).cpu()
    assert out[0, 1].isnan().all() and out[0, 0].isfinite().all()
    cache[1][0, 1, 0, 5] = 127
    q[0, 0, 0, 3] = math.nan
    q[0, 1, 0, 3] = math.inf
    out = tp.cache_attention(q.to(device), *cache).cpu()
    assert out[0, :, 0].isnan().all() and out[0, :, 1:].isfinite().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 1e-46])
def test_scales(device, dtype, n, scale):
    attend(device, rows(1, 2, n, 40, 1, dtype), 1, 2, 80, 40, 4, scale=scale)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scores_that_rise_and_fall_far(device, dtype):
    """Running maxima that move by thousands of units, both ways, in every order of the keys."""
    b, h, m, d = 1, 2, 512, 32
    q = torch.ones(b, h, 1, d, dtype=dtype)
    steps = torch.cat([torch.arange(256.0), torch.arange(256.0).flip(0)]) * 8
    for order in (steps, steps.flip(0) * -1, steps[torch.randperm(m, generator=gen(1))]):
        cache = tp.quantized_cache(b, h, m, d, bits=8, device=device)
        key = order.view(1, 1, m, 1).expand(b, h, m, d).contiguous()
        value = rows(b, h, m, d, 2)
        tp.cache_write_(*cache, key.to(device), value.to(device), torch.zeros(b, dtype=torch.long, device=device))
        cpu = [raw(x) for x in cache]
        k, there = ref.whole(cpu[0], cpu[1], 8, d)
        v, _ = ref.whole(cpu[2], cpu[3], 8, d)
        o, tol = ref.reference(q, k, v, there)
        assert_close(tp.cache_attention(q.to(device), *cache), o, rtol=0.0, atol=tol + TINY)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("width", [(64, 64), (128, 96), (50, 128), (160, 224), (256, 256)], ids=str)
@pytest.mark.parametrize("n", [1, 8, 9, 16])
def test_few_rows_over_short_and_partial_caches(device, dtype, bits, width, n):
    """1 to 32 rows a key head, 16 to 144 keys, with and without added values, holes in the pages."""
    d, dv = width
    for m in (16, 48, 144):
        for mask in (None, torch.randn(n, m, generator=gen(m))):
            attend(device, rows(1, 4, n, d, 1, dtype), 1, 2, m, dv, bits, mask, causal=True, what=f"{m}")
        pages = torch.randperm(m // 16 + 1, generator=gen(m))[:m // 16].view(1, -1)
        pages[0, m // 32] = -1 if m > 16 else 0
        attend(device, rows(1, 4, n, d, 1, dtype), m // 16 + 1, 2, m, dv, bits, pages=pages,
               lengths=torch.tensor([m - 5]), what=f"{m} in pages")


@pytest.mark.parametrize("device", DEVICES)
def test_queries_of_any_layout(device):
    b, h, hk, n, m, d = 2, 4, 2, 3, 48, 50
    cpu, cache = filled(b, hk, m, d, d, 4, device)
    k, there = ref.whole(cpu[0], cpu[1], 4, d)
    v, _ = ref.whole(cpu[2], cpu[3], 4, d)
    base = torch.randn(b, h, n, 2 * d + 3, generator=gen(1))
    for n1 in (1, n):
        for q in (base[:, :, :n1, 1:d + 1], base[:, :, :n1, :2 * d:2], base[:, :1, :n1, :d].expand(b, h, n1, d)):
            o, tol = ref.reference(q, k, v, there)
            on = torch.as_strided(base.to(device), q.shape, q.stride(), q.storage_offset())
            assert_close(tp.cache_attention(on, *cache), o, rtol=0.0, atol=tol + TINY)


def far_apart(x, dim, stride):
    """x's values in a view whose entries along `dim` lie `stride` bytes apart."""
    strides = list(x.stride())
    strides[dim] = stride
    y = torch.zeros(sum((s - 1) * st for s, st in zip(x.shape, strides)) + 1, dtype=torch.uint8, device=x.device)
    return y.as_strided(x.shape, strides).view(x.dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("side", ["key", "value"])
@pytest.mark.parametrize("far", ["codes", "scales"])
def test_rows_and_scales_that_lie_far_apart(device, bits, side, far):
    """Strides over rows past 8 MiB and over blocks past 256 MiB: written, read back, attended to by few rows and
    by many."""
    hk, m, d = 1, 16, 64
    cache = list(tp.quantized_cache(1, hk, m, d, bits=bits, device=device))
    at = 2 * (side == "value") + (far == "scales")
    cache[at] = far_apart(cache[at], 2, (1 << 23) + 16 if far == "codes" else (1 << 28) + 16)
    x = [rows(1, hk, m, d, 50 + k) for k in (0, 1)]
    tp.cache_write_(*cache, *(y.to(device) for y in x), torch.zeros(1, dtype=torch.long, device=device))
    k, v = (ref.decode(*ref.encode(y, bits), bits, d) for y in x)
    got = tp.cache_read(*cache, dtype=F32)
    assert_equal(got[0], k.float())
    assert_equal(got[1], v.float())
    for n in (1, 3, 20, 40):
        for dtype in (F32, BF16):
            q = rows(1, 2, n, d, 60 + n, dtype)
            o, tol = ref.reference(q, k, v, torch.ones(1, m, dtype=torch.bool), causal=True)
            out = tp.cache_attention(q.to(device), *cache, causal=True)
            assert_close(out, o, rtol=0.0, atol=tol + TINY, what=f"{n} {dtype}")


@pytest.mark.parametrize("device", DEVICES)
def test_empty_calls(device):
    for b, n, m in ((0, 1, 16), (2, 0, 16), (2, 1, 0), (2, 3, 0)):
        cache = tp.quantized_cache(b, 2, m, 64, device=device)
        z = torch.zeros(b, 2, n, 64, device=device)
        tp.cache_write_(*cache, z, z, torch.zeros(b, dtype=torch.long, device=device))
        k, v = tp.cache_read(*cache, rows=n)
        assert k.shape == v.shape == (b, 2, n, 64) and not k.any()
        out = tp.cache_attention(torch.ones(b, 4, n, 64, device=device), *cache)
        assert out.shape == (b, 4, n, 64) and not out.any()
    # no pages at all, and tables without entries
    cache = tp.quantized_cache(0, 2, 16, 64, device=device)
    for pages in (torch.zeros(3, 0, dtype=torch.long, device=device), torch.zeros(3, 2, dtype=torch.int32, device=device)):
        z = torch.ones(3, 2, 5, 64, device=device)
        tp.cache_write_(*cache, z, z, torch.zeros(3, dtype=torch.long, device=device), pages=pages)
        assert not tp.cache_read(*cache, rows=5, pages=pages)[0].any()
        assert not tp.cache_attention(z, *cache, pages=pages).any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("paged", [False, True])
def test_tokens_one_by_one_match_one_call(device, dtype, paged):
    """A prompt of ragged lengths, then token by token: written, attended to, and the same as attention over
    what the cache reads back."""
    b, h, hk, d, m, page = 3, 4, 2, 64, 96, 16
    pages = torch.randperm(b * m // page, generator=gen(1)).view(b, -1).int().to(device) if paged else None
    cache = tp.quantized_cache(*((b * m // page, hk, page) if paged else (b, hk, m)), d, device=device)
    lengths = torch.tensor([5, 33, 17], device=device)
    key, value = rows(b, hk, 33, d, 1, dtype, True), rows(b, hk, 33, d, 2, dtype, True)
    tp.cache_write_(*cache, like(key, device), like(value, device), torch.zeros_like(lengths), counts=lengths, pages=pages)
    queries, outs = [], []
    for i in range(20):
        q, k, v = (rows(b, x, 1, d, 10 + 3 * i + y, dtype).to(device) for y, x in enumerate((h, hk, hk)))
        tp.cache_write_(*cache, k, v, lengths, pages=pages)
        lengths = lengths + 1
        queries.append(q)
        outs.append(tp.cache_attention(q, *cache, lengths=lengths, pages=pages))
    k, v = tp.cache_read(*cache, dtype=F32, counts=lengths, pages=pages)
    q = torch.cat(queries, 2)
    want = tp.attention(q.float(), k, v, causal=True, lengths=lengths)
    chunk = tp.cache_attention(q, *cache, causal=True, lengths=lengths, pages=pages)
    # want is off by at most the bound of tests/_cache.py in float32; the outputs by that of their own type
    kc, there = k.cpu().double(), torch.ones(b, m, dtype=torch.bool)
    o, tol = ref.reference(q.cpu(), kc, v.cpu().double(), there, causal=True, lengths=lengths.cpu())
    _, more = ref.reference(q.cpu().float(), kc, v.cpu().double(), there, causal=True, lengths=lengths.cpu())
    for out in (torch.cat(outs, 2), chunk):
        assert_close(out, want, rtol=0.0, atol=tol + more + TINY)


# ---------------------------------------------------------------- refusals
def test_quantized_cache_refuses():
    for bad in (dict(bits=3), dict(rows=17), dict(heads=0), dict(batch=-1), dict(width=0), dict(width=257), dict(value_width=300)):
        args = {**dict(batch=1, heads=1, rows=16, width=32), **bad}
        with pytest.raises(ValueError, match="quantized_cache"):
            tp.quantized_cache(**args)
    kc, ks, vc, vs = tp.quantized_cache(2, 3, 32, 50, 100, bits=8)
    assert kc.dtype == F8 and kc.shape == (2, 3, 32, 64) and vc.shape == (2, 3, 32, 128)
    assert ks.shape == (2, 3, 2, 32) and vs.shape == (2, 3, 4, 32) and ks.dtype == torch.uint8


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    b, h, m, d = 2, 2, 32, 64
    cache = tp.quantized_cache(b, h, m, d, device=device)
    kc, ks, vc, vs = cache
    x = torch.zeros(b, h, 3, d, device=device)
    s = torch.zeros(b, dtype=torch.long, device=device)
    pages = torch.zeros(b, 2, dtype=torch.int32, device=device)

    def refuse(match, f, *args, **kwargs):
        with pytest.raises((RuntimeError, NotImplementedError), match=match):
            f(*args, **kwargs)

    for f, more in ((tp.cache_write_, (x, x, s)), (tp.cache_read, ())):
        refuse("uint8 .4 bits. or float8", f, kc.short(), ks, vc, vs, *more)
        refuse("differ in dtype", f, kc, ks, torch.cat([vc, vc], -1).view(F8), vs, *more)
        refuse("scales must be uint8", f, kc, ks.char(), vc, vs, *more)
        refuse("4-D", f, kc[0], ks, vc, vs, *more)
        refuse("scales must have shape", f, kc, ks[:, :, :1], vc, vs, *more)
        refuse("differ in shape", f, kc, ks, vc[:, :1], vs[:, :1], *more)
        refuse("multiples of 16", f, kc[:, :, :8], ks[..., :8], vc[:, :, :8], vs[..., :8], *more)
        refuse("blocks of 16 bytes", f, kc[..., :24], ks, vc, vs, *more)
        refuse("dense in the last", f, torch.cat([kc, kc], -1)[..., ::2], ks, vc, vs, *more)
        refuse("strides in multiples of 16", f, torch.cat([kc, kc[..., :8]], -1)[..., :32], ks, vc, vs, *more)
        refuse("int32 or int64", f, *cache, *more, pages=pages.short())
        refuse(r"pages must have shape|batch_size", f, *cache, *more, pages=pages[0])
        refuse("counts must have shape", f, *cache, *more, counts=s[:1])
        refuse("counts must be int64 or int32", f, *cache, *more, counts=s.float())
        three = [y[:, :, :48] if i % 2 == 0 else y[..., :48] for i, y in enumerate(tp.quantized_cache(b, h, 64, d, device=device))]
        refuse("power of two", f, *[y.contiguous() for y in three], *more, pages=pages)
    refuse("expected 4-D key", tp.cache_write_, *cache, x[0], x[0], s)
    refuse("dtypes differ", tp.cache_write_, *cache, x, x.bfloat16(), s)
    refuse("supports float32 and bfloat16", tp.cache_write_, *cache, x.half(), x.half(), s)
    refuse("heads", tp.cache_write_, *cache, x[:, :1], x[:, :1], s)
    refuse("do not match", tp.cache_write_, *cache, x, x[:, :, :2], s)
    refuse("do not fill", tp.cache_write_, *cache, x[..., :32], x, s)
    refuse("holds 2 sequences", tp.cache_write_, *cache, x[:1], x[:1], s[:1])
    refuse("starts must have shape", tp.cache_write_, *cache, x, x, s[:1])
    refuse("single memory location|internal", tp.cache_write_, kc[:1].expand(b, h, m, d // 2), ks, vc, vs, x, x, s)
    refuse("no gradient", tp.cache_write_, *cache, x.clone().requires_grad_(), x, s)
    refuse("supports float32 and bfloat16", tp.cache_read, *cache, dtype=torch.half)
    refuse("features of a cache", tp.cache_read, *cache, key_width=65)
    refuse("invalid number of rows", tp.cache_read, *cache, rows=-1)
    f = tp.cache_attention
    refuse("4-D query", f, x[0], *cache)
    refuse("supports float32 and bfloat16", f, x.half(), *cache)
    refuse("supports float32 and bfloat16", f, x.double(), *cache)
    refuse("multiple of the number of key heads", f, x[:, :1], *cache)
    refuse("queries of 32 features", f, x[..., :32], *cache)
    refuse("value_width 20", f, x, *cache, value_width=20)
    wide = tp.quantized_cache(b, h, m, d, 128, device=device)
    refuse("value_width is needed", f, x, *wide)
    refuse("does not broadcast", f, x, *cache, torch.zeros(3, 31, device=device))
    refuse("mask must be bool", f, x, *cache, torch.zeros(3, m, dtype=torch.long, device=device))
    refuse("lengths must have shape", f, x, *cache, lengths=s[:1])
    refuse("scale must be finite", f, x, *cache, scale=math.nan)
    refuse("no gradient", f, x.clone().requires_grad_(), *cache)
    refuse("no gradient", f, x, *cache, torch.zeros(3, m, device=device).requires_grad_())
    with forward_ad.dual_level():
        refuse("forward-mode", f, forward_ad.make_dual(x.clone(), x), *cache)
        refuse("forward-mode", tp.cache_write_, *cache, forward_ad.make_dual(x.clone(), x), x, s)
    with torch.no_grad():  # nothing is asked for
        f(x.clone().requires_grad_(), *cache)
    if device == "cuda":
        refuse("different devices|another device|same device", tp.cache_write_, *cache, x.cpu(), x.cpu(), s)
        refuse("another device|same device", f, x, *cache, lengths=s.cpu())


@pytest.mark.parametrize("device", DEVICES)
def test_writing_refuses_tensors_that_share_memory(device):
    kc, ks, vc, vs = tp.quantized_cache(2, 2, 32, 64, device=device)
    x, s = torch.zeros(2, 2, 3, 64, device=device), torch.zeros(2, dtype=torch.long, device=device)
    inside = vc.view(-1)[:768].view(torch.bfloat16).view(2, 2, 3, 32)
    for cache in ((kc, ks, kc, vs), (kc, ks, vc, ks)):
        with pytest.raises(RuntimeError, match="overlap|single memory|refer"):
            tp.cache_write_(*cache, x, x, s)
    narrow = tp.quantized_cache(2, 2, 32, 32, device=device)
    with pytest.raises(RuntimeError, match="overlap|single memory|refer"):
        tp.cache_write_(narrow[0], narrow[1], vc, vs, inside, x.bfloat16(), s)
    # side by side in one allocation is fine, and so is reading keys as values
    both = torch.zeros(2, 2, 2, 32, 32, dtype=torch.uint8, device=device)
    tp.cache_write_(both[0], ks, both[1], vs, x, x + 1, s)
    both = both.permute(1, 0, 2, 3, 4).contiguous().permute(1, 0, 2, 3, 4)
    tp.cache_write_(both[0], ks, both[1], vs, x, x + 1, s)
    k, v = tp.cache_read(both[1], vs, both[1], vs, dtype=F32, rows=3)
    assert_equal(k, v)
    assert (k == 1).all()


@pytest.mark.parametrize("device", DEVICES)
def test_writing_marks_the_cache_as_changed(device):
    cache = tp.quantized_cache(1, 1, 16, 32, device=device)
    x = torch.ones(1, 1, 1, 32, device=device)
    before = [t._version for t in cache]
    tp.cache_write_(*cache, x, x, torch.zeros(1, dtype=torch.long, device=device))
    assert all(t._version > v for t, v in zip(cache, before))


def test_c_entries_refuse():
    """Errors of the C entries, before anything is launched."""
    lib = capi.lib()

    def desc(**more):
        d = capi.CacheDesc(bits=4, first=1, heads=1, rows=16, key_blocks=1, value_blocks=1, key_codes=4096, key_scales=4096,
                           value_codes=4096, value_scales=4096)
        for side in ("key", "value"):
            getattr(d, side + "_code_strides")[:] = [256, 256, 16]
            getattr(d, side + "_scale_strides")[:] = [16, 16, 16]
        for k, v in more.items():
            setattr(d, k, v)
        return d

    three = (C.c_int64 * 3)(32, 32, 32)

    def write(d, dtype=0, batch=1, n=1, key=4096, width=32, f=lib.tpw_cache_write):
        return f(None if d is None else C.byref(d), dtype, batch, n, key, width, three, 4096, 32, three, None, None, None)

    for f in (lib.tpw_cache_write, lib.tpw_cache_read):
        for bad, text in ((dict(bits=5), b"4 or 8 bits"), (dict(rows=8), b"multiples of 16"), (dict(key_blocks=9), b"blocks"),
                          (dict(value_blocks=0), b"blocks"), (dict(heads=0), b"sizes"), (dict(key_codes=4100), b"16-byte"),
                          (dict(key_scales=0), b"16-byte"), (dict(first=2), b"one entry per sequence"),
                          (dict(rows=48, pages=4096, page_count=1), b"power of two"),
                          (dict(pages=4096, page_count=2 ** 31), b"number of pages"),
                          (dict(rows=1 << 20, pages=4096, page_count=1 << 11), b"too many rows")):
            assert write(desc(**bad), f=f) == 1, bad
            assert text in lib.tpw_last_error(), (bad, lib.tpw_last_error())
        assert write(None, f=f) == 1
        assert write(desc(), dtype=2, f=f) == 1 and b"float32 or bfloat16" in lib.tpw_last_error()
        assert write(desc(), n=-1, f=f) == 1 and write(desc(), width=33, f=f) == 1 and write(desc(), key=None, f=f) == 1
        assert write(desc(first=0), batch=0, f=f) == 0 and write(desc(), n=0, f=f) == 0  # nothing to do

    def attention(**more):
        a = capi.AttentionDesc(dtype=0, batch=1, heads=1, key_heads=1, n=1, m=16, d=32, dv=32, scale=1.0, query=4096, out=4096)
        a.query_strides[:] = a.out_strides[:] = [32, 32, 32]
        for k, v in more.items():
            setattr(a, k, v)
        return a

    for bad, text in ((dict(stats=4096), b"no backward"), (dict(key_heads=0), b"key_heads"), (dict(m=32), b"m differs"),
                      (dict(d=33), b"wider"), (dict(query=None), b"null operand"), (dict(mask_type=1), b"null mask"),
                      (dict(heads=2, key_heads=2), b"cache's heads"), (dict(scale=math.inf), b"scale")):
        a = attention(**bad)
        assert lib.tpw_cache_attention(C.byref(a), C.byref(desc()), None, None) == 1, bad
        assert text in lib.tpw_last_error(), (bad, lib.tpw_last_error())
    a = attention(m=4096)
    d = desc(rows=4096)
    assert lib.tpw_cache_attention_workspace_size(C.byref(a), C.byref(d)) > 0
    assert lib.tpw_cache_attention(C.byref(a), C.byref(d), None, None) == 1 and b"workspace" in lib.tpw_last_error()
    assert lib.tpw_cache_attention_workspace_size(None, None) == 0
    a = attention(batch=0)
    assert lib.tpw_cache_attention(C.byref(a), C.byref(desc(first=0)), None, None) == 0
    # more blocks than a launch has room for
    for f in (lib.tpw_cache_write, lib.tpw_cache_read):
        assert write(desc(first=1 << 24), batch=1 << 24, f=f) == 1 and b"too many" in lib.tpw_last_error()
        assert write(desc(heads=1 << 62), f=f) == 1 and b"too many" in lib.tpw_last_error()
    a = attention(batch=1 << 24)
    assert lib.tpw_cache_attention(C.byref(a), C.byref(desc(first=1 << 24)), None, None) == 1
    assert b"too many" in lib.tpw_last_error()


def c_cache(**more):
    """A descriptor of one sequence of one head, 16 rows of a block, at addresses that nothing is read from."""
    d = capi.CacheDesc(bits=4, first=1, heads=1, rows=16, key_blocks=1, value_blocks=1, key_codes=4096, key_scales=4096,
                       value_codes=4096, value_scales=4096)
    for side in ("key", "value"):
        getattr(d, side + "_code_strides")[:] = [256, 256, 16]
        getattr(d, side + "_scale_strides")[:] = [16, 16, 16]
    for k, v in more.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("dtype", [capi.TPW_F32, capi.TPW_BF16])
@pytest.mark.parametrize("d", [1, 50, 64, 90, 200])
def test_workspace_sizes_before_and_after_there_are_operands(dtype, d):
    """A query without an address counts as an aligned one: rows that have to be copied are counted."""
    lib, blocks = capi.lib(), ref.blocks_of(d)
    for n, m, mask_type in ((1, 16, 0), (1, 1008, 1), (70, 1008, 2), (1000, 1008, 0), (1000, 1008, 1)):
        c = c_cache(first=2, heads=2, rows=m, key_blocks=blocks, value_blocks=blocks)
        sizes = []
        for address in (None, 4096):
            a = capi.AttentionDesc(dtype=dtype, batch=2, heads=4, key_heads=2, n=n, m=m, d=d, dv=d, scale=1.0,
                                   mask_type=mask_type, query=address, out=address, mask=address, lengths=address)
            a.query_strides[:] = a.out_strides[:] = [4 * n * d, n * d, d]
            a.mask_strides[:] = [0, 0, m, 1]
            sizes.append(lib.tpw_cache_attention_workspace_size(C.byref(a), C.byref(c)))
        assert sizes[0] == sizes[1], (n, m, mask_type, sizes)
        # the copy of the query alone: keys and values have no addresses here, and need no copies
        copied = 2 * 4 * n * -(-d * (4 if dtype == capi.TPW_F32 else 2) // 16) * 16
        assert sizes[0] >= copied or d % 8 == 0 or n == 1


def test_c_entries_take_rows_and_scales_far_apart():
    """What a descriptor may hold, seen by calls of no rows."""
    lib, three = capi.lib(), (C.c_int64 * 3)(32, 32, 32)
    for row, block, rc in ((1 << 40, 1 << 40, 0), (-16, 16, 1), (16, -16, 1), (24, 16, 1), (16, 24, 1)):
        c = c_cache(key_blocks=2, value_blocks=2)
        for side in ("key", "value"):
            getattr(c, side + "_code_strides")[:] = [0, 0, row]
            getattr(c, side + "_scale_strides")[:] = [0, 0, block]
        for f in (lib.tpw_cache_write, lib.tpw_cache_read):
            assert f(C.byref(c), 0, 1, 0, 4096, 32, three, 4096, 32, three, None, None, None) == rc, (row, block)


def test_c_workspace_of_tables_without_pages():
    """Sizes of a call over no keys: what a mask over them would take is not asked for."""
    lib = capi.lib()
    for dtype in (capi.TPW_F32, capi.TPW_BF16):
        for n in (1, 100):
            sizes = []
            for mask_type in (0, 1, 2):
                a = capi.AttentionDesc(dtype=dtype, batch=2, heads=4, key_heads=2, n=n, m=64, d=90, dv=90, scale=1.0,
                                       mask_type=mask_type)
                a.query_strides[:] = a.out_strides[:] = [4 * n * 90, n * 90, 90]
                c = c_cache(first=0, heads=2, key_blocks=3, value_blocks=3, pages=4096, page_count=4, page_pitch=4)
                sizes.append(lib.tpw_cache_attention_workspace_size(C.byref(a), C.byref(c)))
            assert sizes[0] == sizes[1] == sizes[2], (dtype, n, sizes)


# ---------------------------------------------------------------- on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 8, 60])
def test_results_repeat_bit_for_bit(n):
    _, cache = filled(2, 2, 4096, 128, 128, 4, "cuda")
    q = rows(2, 8, n, 128, 1, BF16).cuda()
    outs = [tp.cache_attention(q, *cache, causal=True) for _ in range(3)]
    for o in outs[1:]:
        assert_equal(o, outs[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 100])
@pytest.mark.parametrize("mask_type", [0, 1, 2])
def test_c_entry_over_tables_without_pages(dtype, n, mask_type):
    """Tables over no pages at all, called through the C entry: zeros, whatever the mask."""
    b, h, hk, d = 2, 4, 2, 90  # rows that are copied first
    q, pages = rows(b, h, n, d, 1, dtype).cuda(), torch.zeros(b, 4, dtype=torch.int32, device="cuda")
    out, mask = torch.full_like(q, 7.0), torch.ones(n, 64, dtype=torch.bool if mask_type == 1 else F32, device="cuda")
    a = capi.AttentionDesc(dtype=capi.TPW_F32 if dtype == F32 else capi.TPW_BF16, batch=b, heads=h, key_heads=hk, n=n, m=64,
                           d=d, dv=d, scale=1.0, mask_type=mask_type, query=q.data_ptr(), out=out.data_ptr(),
                           mask=mask.data_ptr())
    a.query_strides[:] = a.out_strides[:] = q.stride()[:3]
    a.mask_strides[:] = [0, 0, 64, 1]
    c = c_cache(first=0, heads=hk, key_blocks=3, value_blocks=3, key_codes=None, key_scales=None, value_codes=None,
                value_scales=None, pages=pages.data_ptr(), page_count=4, page_pitch=4)
    size = capi.lib().tpw_cache_attention_workspace_size(C.byref(a), C.byref(c))
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    capi.call("tpw_cache_attention", C.byref(a), C.byref(c), ws.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert not out.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [1, 12, 100])
def test_c_entry_with_fewer_features_than_the_cache(dtype, bits, n):
    """Blocks behind the features of a call are no part of it, whatever they hold."""
    h, hk, m, d = 4, 2, 48, 30
    cpu, cache = filled(1, hk, m, 100, 70, bits, "cuda")
    cache[1][:, :, 1:] = 255
    cache[3][:, :, 1:] = 255
    q = rows(1, h, n, d, 1, dtype).cuda()
    out = torch.full_like(q, 7.0)
    a = capi.AttentionDesc(dtype=capi.TPW_F32 if dtype == F32 else capi.TPW_BF16, batch=1, heads=h, key_heads=hk, n=n, m=m,
                           d=d, dv=d, scale=1.0, query=q.data_ptr(), out=out.data_ptr())
    a.query_strides[:] = a.out_strides[:] = q.stride()[:3]
    c = c_cache(bits=bits, heads=hk, rows=m, key_blocks=4, value_blocks=3, **{
        f"{side}_{what}": cache[2 * k + i].data_ptr()
        for k, side in enumerate(("key", "value")) for i, what in enumerate(("codes", "scales"))})
    for k, side in enumerate(("key", "value")):
        getattr(c, side + "_code_strides")[:] = cache[2 * k].stride()[:3]
        getattr(c, side + "_scale_strides")[:] = cache[2 * k + 1].stride()[:3]
    size = capi.lib().tpw_cache_attention_workspace_size(C.byref(a), C.byref(c))
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    capi.call("tpw_cache_attention", C.byref(a), C.byref(c), ws.data_ptr(), torch.cuda.current_stream().cuda_stream)
    k, there = ref.whole(cpu[0], cpu[1], bits, d)
    v, _ = ref.whole(cpu[2], cpu[3], bits, d)
    o, tol = ref.reference(q.cpu(), k, v, there, scale=1.0)
    assert_close(out, o, rtol=0.0, atol=tol + TINY)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,m", [(1, 8208), (1, 40912), (5, 24704), (20, 24704), (40, 24704)])
@pytest.mark.parametrize("d", [64, 160])
def test_one_head_over_a_long_cache(dtype, n, m, d):
    """More chunks of keys than there may be parts."""
    attend("cuda", rows(1, 1, n, d, 3, dtype), 1, 1, m, d, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("bits,d", [(4, 64), (4, 128), (4, 250), (8, 128), (8, 250)])
@pytest.mark.parametrize("m", [240, 1024, 1104])
def test_short_caches_of_many_heads(dtype, bits, d, m):
    """Up to a length one block works on a sequence and head; past it several, whose parts are joined."""
    lengths = torch.tensor([m - k * m // 15 for k in range(16)])
    attend("cuda", rows(16, 16, 1, d, 80, dtype), 16, 8, m, d, bits, lengths=lengths)


@pytest.mark.gpu
def test_graphs_and_streams():
    """A token's write and attention captured twice, replayed in turn with eager work between; and the same on
    a stream of its own."""
    b, h, hk, m, d = 2, 8, 2, 512, 64
    cache = tp.quantized_cache(b, hk, m, d, device="cuda")
    other = tp.quantized_cache(b, hk, m, d, device="cuda")
    eager = tp.quantized_cache(b, hk, m, d, device="cuda")
    q, k, v = rows(b, h, 1, d, 1).cuda(), rows(b, hk, 1, d, 2).cuda(), rows(b, hk, 1, d, 3).cuda()
    lengths = torch.zeros(b, dtype=torch.long, device="cuda")

    def step(c, at):
        tp.cache_write_(*c, k, v, at)
        return tp.cache_attention(q, *c, lengths=at + 1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up
        step(cache, lengths)
        step(other, lengths)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for c in (cache, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(c, lengths))
        graphs.append(g)
    for i in range(6):
        for x, s in ((q, 20), (k, 40), (v, 60)):
            x.copy_(rows(*x.shape[:3], d, s + i))
        for g in graphs:
            g.replay()
        want = step(eager, lengths)
        for o in outs:
            assert_equal(o, want)
        lengths += 1
        torch.cuda.synchronize()
    for c in (cache, other):
        for x, y in zip(c, eager):
            assert_equal(raw(x)[:, :, :6] if x.shape[2] == m else raw(x)[..., :6],
                         raw(y)[:, :, :6] if y.shape[2] == m else raw(y)[..., :6])
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        mine = step(eager, lengths)
    side.synchronize()
    assert_equal(mine, step(eager, lengths))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_long_caches(bits):
    """Many parts, a ragged batch, against the oracle."""
    attend("cuda", rows(2, 8, 1, 128, 1, BF16), 2, 2, 8192, 128, bits, lengths=torch.tensor([8191, 5003]))
    attend("cuda", rows(2, 8, 2, 64, 1), 2, 2, 8192, 64, bits, causal=True, lengths=torch.tensor([8190, 77]))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Codes of 4.3 GB a side: rows written, read and attended to behind 2^32 bytes."""
    m, d = (1 << 24) + 4096, 256
    cache = tp.quantized_cache(1, 1, m, d, bits=8, device="cuda")
    n = 100
    start = torch.tensor([m - n], device="cuda")
    key, value = rows(1, 1, n, d, 1), rows(1, 1, n, d, 2)
    tp.cache_write_(*cache, key.cuda(), value.cuda(), start)
    codes, scales = ref.encode(key, 8)
    assert_equal(raw(cache[0][:, :, m - n:]), codes)
    want = ref.decode(*ref.encode(value, 8), 8, d)
    assert_equal(tp.cache_read(*cache, dtype=F32, starts=start, rows=n)[1], want.float())
    # all but the last keys score 0 and weigh exp(0 - top), their values are 0: drown them out
    k = ref.decode(codes, scales, 8, d)
    for rows_ in (1, 40):
        q = (key[:, :, -1:].expand(1, 1, rows_, d) * 0.5).contiguous()
        s = 0.5 * (key[0, 0, -1].double() @ k[0, 0].T)
        assert s.max() > 60  # exp(-60) 2^24 < 1e-18
        mask = torch.full((1, m), -math.inf, device="cuda")
        mask[0, m - n:] = 0.0
        o, tol = ref.reference(q, k, want, torch.ones(1, n, dtype=torch.bool), scale=1.0)
        out = tp.cache_attention(q.cuda(), *cache, scale=1.0)
        assert_close(out, o, rtol=0.0, atol=tol + 1e-15)
        out = tp.cache_attention(q.cuda(), *cache, mask, scale=1.0)
        assert_close(out, o, rtol=0.0, atol=tol + TINY)

"""attention and rotary_embedding: forward, gradients, masks, lengths, layouts and refusals, against
the plain 64-bit forms of tests/_attention.py with bounds derived there."""
import ctypes as C
import math
import subprocess
import sys
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import torchpairwise as tp
from torchpairwise_amd import _capi as capi
from tests._attention import reference, rotate
from tests._util import assert_close, assert_equal, gen, randn

F32, BF16 = torch.float32, torch.bfloat16
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
TINY = 1e-30


def rows(b, h, n, d, seed, dtype=F32, rows_first=False):
    x = torch.randn(b, n, h, d, generator=gen(seed)) if rows_first else torch.randn(b, h, n, d, generator=gen(seed))
    x = x.to(dtype)
    return x.transpose(1, 2) if rows_first else x


def on(device, *xs):
    """Copies on the device with the same strides."""
    out = []
    for x in xs:
        if x is None:
            out.append(None)
            continue
        y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=device)
        y.copy_(x)
        out.append(y)
    return out


def check(device, q, k, v, mask=None, causal=False, scale=None, lengths=None, grad=None, what=""):
    want = reference(q, k, v, mask, causal, scale, lengths, grad)
    dq, dk, dv, dm, dl, dg = on(device, q, k, v, None, lengths, grad)
    dm = None if mask is None else mask.to(device)
    if grad is not None:
        for x in (dq, dk, dv):
            x.requires_grad_()
    out = tp.attention(dq, dk, dv, dm, causal=causal, scale=scale, lengths=dl)
    assert out.dtype == q.dtype and out.shape == (*q.shape[:-1], v.shape[-1])
    assert_close(out, want["out"], rtol=0.0, atol=want["tol_out"] + TINY, what=f"{what} out")
    if grad is None:
        return out
    grads = torch.autograd.grad(out, (dq, dk, dv), dg)
    for name, g, x in zip(("dq", "dk", "dv"), grads, (q, k, v)):
        assert g.dtype == x.dtype and g.shape == x.shape
        assert_close(g, want[name], rtol=0.0, atol=want["tol_" + name] + TINY, what=f"{what} {name}")
    return out, grads


# b, heads, key heads, n, m, d, dv, rows first
SIZES = [
    (1, 1, 1, 1, 1, 1, 1, False),
    (1, 2, 1, 1, 7, 8, 8, False),
    (2, 3, 3, 5, 33, 50, 50, True),
    (1, 4, 2, 31, 64, 64, 64, False),
    (2, 4, 1, 65, 129, 96, 96, True),
    (1, 2, 2, 128, 128, 128, 128, False),
    (1, 6, 2, 130, 257, 128, 128, True),
    (3, 2, 2, 70, 40, 80, 16, False),
    (1, 2, 1, 100, 75, 33, 200, True),
    (1, 2, 2, 97, 161, 256, 256, False),
    (1, 2, 1, 64, 100, 203, 256, True),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward_and_gradients(device, dtype, causal, size):
    b, h, hk, n, m, d, dv, rf = size
    check(device, rows(b, h, n, d, 1, dtype, rf), rows(b, hk, m, d, 2, dtype, rf), rows(b, hk, m, dv, 3, dtype, rf),
          causal=causal, grad=rows(b, h, n, dv, 4, dtype, rf))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [64, 90, 128, 256])
@pytest.mark.parametrize("kind", ["keep", "keep_keys", "bias", "bias_heads", "bias_bf16", "keep_strided"])
def test_masks(device, dtype, d, kind):
    b, h, hk, n, m = 2, 4, 2, 45, 91
    g = gen(7)
    if kind == "keep":
        mask = torch.rand(n, m, generator=g) < 0.4
        mask[3] = False  # a row that nothing is left to
        mask[40:] = False
        mask[5] = torch.arange(m) == 17  # one key
    elif kind == "keep_keys":
        mask = (torch.rand(b, 1, 1, m, generator=g) < 0.5)
        mask[1] = False
    elif kind == "keep_strided":
        mask = (torch.rand(b, h, m, n, generator=g) < 0.5).mT
    elif kind == "bias":
        mask = torch.randn(n, m, generator=g)
        mask[torch.rand(n, m, generator=g) < 0.3] = -math.inf
        mask[2] = -math.inf
        mask[4] = torch.finfo(torch.float32).min  # the lowest value: every key weighs the same
        mask[6, 1:] = torch.finfo(torch.float32).min
    elif kind == "bias_heads":
        mask = torch.randn(h, 1, m, generator=g) * 3
    else:
        mask = torch.randn(1, h, n, m + 1, generator=g).to(BF16)[..., 1:]
    check(device, rows(b, h, n, d, 1, dtype), rows(b, hk, m, d, 2, dtype), rows(b, hk, m, d, 3, dtype), mask,
          grad=rows(b, h, n, d, 4, dtype), what=kind)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths_and_what_lies_behind_them(device, dtype, causal):
    """Lengths of 0 and 1, past m and below 0; rows behind them hold NaN and infinities and are not
    read; their gradients are zeros."""
    b, h, hk, n, m, d = 6, 2, 1, 9, 150, 64
    lengths = torch.tensor([0, 1, 64, 149, 999, -5])
    q, k, v = rows(b, h, n, d, 1, dtype), rows(b, hk, m, d, 2, dtype), rows(b, hk, m, d, 3, dtype)
    for i, l in enumerate(lengths.clamp(0, m).tolist()):
        k[i, :, l:] = math.nan
        v[i, :, l:] = math.inf
    out, (dq, dk, dv) = check(device, q, k, v, causal=causal, lengths=lengths, grad=rows(b, h, n, d, 4, dtype))
    for i in (0, 5):
        for x in (out, dq, dk, dv):
            assert not x[i].any()
    assert not dk[1, :, 1:].any() and not dv[2, :, 64:].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("additive", [False, True])
def test_keys_that_a_mask_leaves_out_may_score_nan(device, dtype, additive):
    b, h, n, m, d = 1, 2, 40, 70, 64
    q, k, v = rows(b, h, n, d, 1, dtype), rows(b, h, m, d, 2, dtype), rows(b, h, m, d, 3, dtype)
    off = torch.zeros(m, dtype=torch.bool)
    off[[0, 33, 69]] = True
    mask = torch.where(off, -math.inf, 0.0).expand(n, m) if additive else ~off.expand(n, m)
    want = reference(q, k, v, mask)
    k = k.clone()
    k[:, :, 0] = math.nan
    k[:, :, 33] = math.inf
    k[:, :, 69] = -math.inf
    out = tp.attention(*on(device, q, k, v), mask.to(device))
    assert_close(out, want["out"], rtol=0.0, atol=want["tol_out"])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_keys_behind_the_causal_limit_may_score_nan(device, dtype):
    n, d = 150, 64
    q, k, v = rows(1, 2, n, d, 1, dtype), rows(1, 2, n, d, 2, dtype), rows(1, 2, n, d, 3, dtype)
    want = reference(q, k, v, causal=True)
    k = k.clone()
    k[:, :, 70], k[:, :, 140] = math.inf, math.nan
    out = tp.attention(*on(device, q, k, v), causal=True).cpu()
    assert_close(out[:, :, :70], want["out"][:, :, :70], rtol=0.0, atol=want["tol_out"][:, :, :70])
    assert out[:, :, 140:].isnan().all()


@pytest.mark.parametrize("device", DEVICES)
def test_nan_and_infinite_scores_stay_in_their_row(device):
    q, k, v = rows(1, 1, 40, 64, 1), rows(1, 1, 70, 64, 2), rows(1, 1, 70, 64, 3)
    want = reference(q, k, v)
    q[0, 0, 3, 5] = math.nan
    out = tp.attention(*on(device, q, k, v)).cpu()
    assert out[0, 0, 3].isnan().all()
    others = torch.arange(40) != 3
    assert_close(out[:, :, others], want["out"][:, :, others], rtol=0.0, atol=want["tol_out"][:, :, others])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 3.0])
def test_scales(device, dtype, scale):
    check(device, rows(1, 2, 33, 40, 1, dtype), rows(1, 2, 65, 40, 2, dtype), rows(1, 2, 65, 40, 3, dtype), scale=scale,
          grad=rows(1, 2, 33, 40, 4, dtype))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [1e-46, -1e-300])
@pytest.mark.parametrize("mask", [None, "keep", "bias"])
def test_scales_below_the_range_of_32_bits(device, scale, mask):
    """The same as a scale of zero: equal weights for the keys that are left, none for the others."""
    if mask == "keep":
        mask = torch.rand(33, 65, generator=gen(5)) < 0.5
    elif mask == "bias":
        mask = randn(33, 65, seed=5).masked_fill(torch.rand(33, 65, generator=gen(6)) < 0.5, -math.inf)
    check(device, rows(1, 2, 33, 40, 1), rows(1, 2, 65, 40, 2), rows(1, 2, 65, 40, 3), mask, causal=True, scale=scale,
          grad=rows(1, 2, 33, 40, 4))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignment(device, dtype):
    """Sliced features (rows not dense), a column offset that breaks 16-byte alignment, transposed
    features, rows a stride apart, broadcast batch and heads, an expanded gradient."""
    b, h, n, m, d = 2, 4, 37, 83, 64
    base = rows(b, h, m, 3 * d + 5, 1, dtype)
    q = rows(b, h, n, d + 3, 2, dtype)[..., 3:]
    grad = rows(b, h, n, d, 4, dtype)
    k, v = base[..., 1:1 + d], base[..., 1 + d:1 + 2 * d]
    check(device, q, k, v, grad=grad, what="offset")
    check(device, rows(b, h, 2 * n, d, 2, dtype)[:, :, ::2], rows(b, h, d, m, 5, dtype).mT, base[..., ::3][..., :d],
          grad=grad, what="strided")
    one = rows(1, 1, m, d, 6, dtype)
    kk = one.expand(b, h, m, d)
    want = reference(q, kk, kk, grad=grad)
    dq, dk, dg = on(device, q, one, grad)
    dk.requires_grad_()
    x = dk.expand(b, h, m, d)
    out = tp.attention(dq, x, x)
    assert_close(out, want["out"], rtol=0.0, atol=want["tol_out"], what="broadcast")
    (got,) = torch.autograd.grad(out, dk, dg)
    tol = (want["tol_dk"] + want["tol_dv"]).sum((0, 1), keepdim=True)
    both = want["dk"] + want["dv"]
    # autograd adds the two and sums over b and h in the data type
    steps = b * h + 2
    tol = tol + steps * torch.finfo(dtype).eps / 2 * both.abs().sum((0, 1), keepdim=True)
    assert_close(got, both.sum((0, 1), keepdim=True), rtol=0.0, atol=tol, what="broadcast gradient")
    ones = torch.ones(1, dtype=dtype).expand(b, h, n, d)
    want = reference(q, k, v, grad=ones)
    leaves = [x.detach().requires_grad_() for x in on(device, q, k, v)]
    got = torch.autograd.grad(tp.attention(*leaves), leaves, torch.ones(1, dtype=dtype, device=device).expand(b, h, n, d))
    for name, x in zip(("dq", "dk", "dv"), got):
        assert_close(x, want[name], rtol=0.0, atol=want["tol_" + name] + TINY, what=f"expanded gradient {name}")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,causal,density", [(32, True, 1.0), (96, True, 1.0), (200, False, 0.02), (20, False, 0.25)])
def test_bf16_gradients_of_rows_on_few_keys(device, n, causal, density):
    """dq and dk of bfloat16 rows that rest on few keys: two roundings of the same size (the scores'
    gradients for the matrix cores, the result) make sqrt(2) of what rounding the exact result costs;
    from a rounded output alone delta would make it up to 1.7."""
    h, d = 16, 64
    mask = torch.rand(n, n, generator=gen(5)) < density
    mask[torch.arange(n), torch.arange(n)] = True
    q, k, v, grad = (rows(1, h, n, d, i, BF16) for i in range(1, 5))
    want = reference(q, k, v, mask, causal, grad=grad)
    leaves = [x.requires_grad_() for x in on(device, q, k, v)]
    got = torch.autograd.grad(tp.attention(*leaves, mask.to(device), causal=causal), leaves, grad.to(device))
    for name, x in zip(("dq", "dk"), got):
        exact = want[name]
        assert (x.cpu().double() - exact).norm() <= 1.5 * (exact.to(BF16).double() - exact).norm(), name


@pytest.mark.parametrize("device", DEVICES)
def test_two_and_three_dimensions(device):
    q, k, v = randn(2, 30, 48, seed=1), randn(2, 50, 48, seed=2), randn(2, 50, 20, seed=3)
    mask = torch.rand(2, 30, 50, generator=gen(4)) < 0.7
    full = tp.attention(q[:, None], k[:, None], v[:, None], mask[:, None])[:, 0]
    for x, got in ((full, tp.attention(*on(device, q, k, v), mask.to(device))),
                   (full[0], tp.attention(*on(device, q[0], k[0], v[0]), mask[0].to(device)))):
        assert got.shape == x.shape
        assert_close(got, x, rtol=1e-4, atol=1e-5)
    for dtype in (F32, BF16):
        x = [y.to(dtype) for y in (q, k, v, randn(2, 30, 20, seed=5))]
        want = reference(*(y[:, None] for y in x[:3]), grad=x[3][:, None])
        for pick in (slice(None), 0, slice(1)):  # 3-D, 2-D, one entry
            leaves = [y[pick].detach().requires_grad_() for y in on(device, *x[:3])]
            got = torch.autograd.grad(tp.attention(*leaves), leaves, x[3][pick].to(device))
            for name, g in zip(("dq", "dk", "dv"), got):
                assert_close(g, want[name][:, 0][pick], rtol=0.0, atol=want["tol_" + name][:, 0][pick] + TINY, what=name)
    shape = tp.attention(*on(device, rows(2, 4, 9, 16, 1, F32, True), rows(2, 2, 9, 16, 2), rows(2, 2, 9, 8, 3)))
    assert shape.transpose(1, 2).is_contiguous()  # rows before heads, as the queries have them


@pytest.mark.parametrize("device", DEVICES)
def test_empty_sizes(device):
    for b, h, n, m in ((0, 2, 3, 4), (2, 0, 3, 4), (2, 2, 0, 4), (2, 2, 3, 0)):
        q = torch.zeros(b, h, n, 8, device=device, requires_grad=True)
        k = torch.ones(b, 2, m, 8, device=device, requires_grad=True)
        v = torch.ones(b, 2, m, 5, device=device, requires_grad=True)
        out = tp.attention(q, k, v)
        assert out.shape == (b, h, n, 5) and not out.any()
        for g, x in zip(torch.autograd.grad(out.sum(), (q, k, v)), (q, k, v)):
            assert g.shape == x.shape and not g.any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [8, 128, 256])
@pytest.mark.parametrize("b,h,n,m", [(0, 2, 3, 4), (2, 0, 3, 4), (2, 2, 0, 4), (2, 2, 3, 0)])
def test_empty_sizes_by_width(device, dtype, d, b, h, n, m):
    q, k, v = (torch.ones(*s, dtype=dtype, device=device, requires_grad=True)
               for s in ((b, h, n, d), (b, 2, m, d), (b, 2, m, d)))
    out = tp.attention(q, k, v)
    assert out.shape == (b, h, n, d) and not out.any()
    for g, x in zip(torch.autograd.grad(out.sum(), (q, k, v)), (q, k, v)):
        assert g.shape == x.shape and not g.any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d", [50, 128])
@pytest.mark.parametrize("b,h,n,m", [(0, 2, 3, 4), (2, 0, 3, 4), (2, 2, 0, 4), (2, 2, 3, 0)])
@pytest.mark.parametrize("kind", ["keep", "bias", "bias_heads"])
def test_empty_sizes_with_masks(device, dtype, d, b, h, n, m, kind):
    mask = {"keep": lambda: torch.ones(n, m, dtype=torch.bool), "bias": lambda: torch.zeros(n, m),
            "bias_heads": lambda: torch.zeros(b, h, n, m)}[kind]().to(device)
    q, k, v = (torch.ones(*s, dtype=dtype, device=device, requires_grad=True)
               for s in ((b, h, n, d), (b, 2, m, d), (b, 2, m, d)))
    out = tp.attention(q, k, v, mask)
    assert out.shape == (b, h, n, d) and not out.any()
    for g, x in zip(torch.autograd.grad(out.sum(), (q, k, v)), (q, k, v)):
        assert g.shape == x.shape and not g.any()


def test_c_entries_ask_for_no_mask_without_queries():
    """A mask over no queries has no address: the entry asks for what comes after the mask.  Nothing is
    launched."""
    lib = capi.lib()
    q, k, v, out = (torch.zeros(1, 2, n, 8) for n in (0, 3, 3, 0))
    for mask_type in (1, 2):
        a = _desc(q, k, v, out, mask_type=mask_type, grad_key=None, grad_value=None)
        # stops at the gradients' addresses, which come after the operands' and before any launch
        assert lib.tpw_attention_backward(C.byref(a), None, None) == 1 and b"null operand" in lib.tpw_last_error()
        gk, gv = torch.zeros_like(k), torch.zeros_like(v)
        a = _desc(q, k, v, out, mask_type=mask_type, grad_key=gk.data_ptr(), grad_value=gv.data_ptr())
        a.grad_key_strides[:] = a.grad_value_strides[:] = k.stride()[:3]
        # the workspace is asked for after the mask
        assert lib.tpw_attention_backward(C.byref(a), None, None) == 1 and b"workspace" in lib.tpw_last_error()


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    q, k, v = (x.to(device) for x in (randn(2, 4, 5, 8, seed=1), randn(2, 2, 6, 8, seed=2), randn(2, 2, 6, 3, seed=3)))
    at = tp.attention

    def refuses(message, *args, **kw):
        with pytest.raises(RuntimeError, match=message):
            at(*args, **kw)

    refuses("2-D, 3-D or 4-D", q[0, 0, 0], k, v)
    refuses("same number of dimensions", q, k[0], v[0])
    refuses("dtypes differ", q, k.to(BF16), v)
    refuses("supports float32 and bfloat16", q.half(), k.half(), v.half())
    refuses("batch_size", q[:1], k, v)
    refuses("feature dimension", q[..., :7], k, v)
    refuses("keys and values", q, k[:, :, :5], v)
    refuses("heads of key and value", q, k, v[:, :1])
    refuses("multiple of the number of key heads", q[:, :3], k, v)
    refuses("1 to 256 features", torch.zeros(1, 1, 2, 257, device=device), torch.zeros(1, 1, 2, 257, device=device),
            torch.zeros(1, 1, 2, 8, device=device))
    refuses("does not broadcast", q, k, v, torch.ones(4, 6, dtype=torch.bool, device=device))
    refuses("mask must be bool", q, k, v, torch.ones(5, 6, dtype=torch.int32, device=device))
    refuses("mask has no gradient", q, k, v, torch.zeros(5, 6, device=device, requires_grad=True))
    refuses("lengths must have shape", q, k, v, lengths=torch.tensor([1], device=device))
    refuses("lengths must be int64", q, k, v, lengths=torch.tensor([1.0, 2.0], device=device))
    refuses("scale must be finite", q, k, v, scale=math.inf)
    leaf = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(at(leaf, k, v).sum(), leaf, create_graph=True)
    x, pos, f = q, torch.arange(5, device=device), torch.ones(4, dtype=torch.float64, device=device)
    for message, args in (("2-D, 3-D or 4-D", (x[0, 0, 0], pos, f)), ("positions must have", (x, pos[:4], f)),
                          ("positions must be int64", (x, pos.float(), f)), ("do not fit", (x, pos, f.repeat(2))),
                          ("frequencies must be", (x, pos, f.long())), ("supports float32", (x.half(), pos, f))):
        with pytest.raises(RuntimeError, match=message):
            tp.rotary_embedding(*args)
    with pytest.raises(RuntimeError, match="scale must be finite"):
        tp.rotary_embedding(x, pos, f, scale=math.nan)
    with pytest.raises(RuntimeError, match="frequencies have no gradient"):
        tp.rotary_embedding(x, pos, f.clone().requires_grad_())


def _desc(q, k, v, out, stats=None, **kw):
    """tpw_attention_desc of dense 4-D rows (C entry)."""
    a = capi.AttentionDesc(dtype=capi.TPW_F32 if q.dtype == F32 else capi.TPW_BF16, batch=q.shape[0], heads=q.shape[1],
                           key_heads=k.shape[1], n=q.shape[2], m=k.shape[2], d=q.shape[3], dv=v.shape[3],
                           scale=q.shape[3] ** -0.5, query=q.data_ptr(), key=k.data_ptr(), value=v.data_ptr(),
                           out=out.data_ptr(), stats=None if stats is None else stats.data_ptr())
    for name, x in (("query", q), ("key", k), ("value", v), ("out", out)):
        getattr(a, name + "_strides")[:] = x.stride()[:3]
    for name, value in kw.items():
        setattr(a, name, value)
    return a


def test_c_entries_refuse_on_the_host():
    """Refusals and workspace sizes need no GPU: nothing is launched."""
    lib = capi.lib()
    q, k, v, out = (torch.zeros(1, 2, 3, 8) for _ in range(4))
    for message, kw in ((b"1 to 256 features", {"d": 0}), (b"1 to 256 features", {"dv": 257}),
                        (b"multiple of key_heads", {"key_heads": 3}), (b"unknown mask type", {"mask_type": 9}),
                        (b"float32 or bfloat16", {"dtype": capi.TPW_F64}), (b"scale must be finite", {"scale": math.inf}),
                        (b"negative size", {"n": -1}), (b"null operand", {"query": None}),
                        (b"null mask", {"mask_type": 1}), (b"too many rows", {"m": 1 << 31})):
        a = _desc(q, k, v, out, **kw)
        assert lib.tpw_attention(C.byref(a), None, None) == 1 and message in lib.tpw_last_error(), message
    a = _desc(q, k, v, out)
    a.key_strides[2] = 4  # rows overlap
    assert lib.tpw_attention(C.byref(a), None, None) == 1 and b"overlap" in lib.tpw_last_error()
    a = _desc(q, k, v, out)
    assert lib.tpw_attention_backward(C.byref(a), None, None) == 1  # gradients missing
    for n, m in ((0, 3), (3, 0), (0, 0), (1, 1), (1, 100000), (5000, 5000)):
        for dtype in (capi.TPW_F32, capi.TPW_BF16):
            for d in (1, 50, 96, 130, 256):
                a = _desc(q, k, v, out, dtype=dtype, n=n, m=m, d=d, dv=d)
                for name in ("query", "key", "value", "out", "grad_out", "grad_query", "grad_key", "grad_value"):
                    getattr(a, name + "_strides")[:] = [d * 5000 * 2, d * 5000, d]
                assert lib.tpw_attention_workspace_size(C.byref(a)) >= 0
                assert lib.tpw_attention_backward_workspace_size(C.byref(a)) >= 4 * 3 * 2 * n
    s = (C.c_int64 * 3)(48, 24, 8)
    assert lib.tpw_rotary(None, capi.TPW_F32, 1, 2, 3, 8, s, None, None, None, 5, 0, 0, 1.0, None, s, None) == 1
    assert lib.tpw_rotary(None, capi.TPW_F64, 1, 2, 3, 8, s, None, None, None, 4, 0, 0, 1.0, None, s, None) == 1
    assert lib.tpw_rotary(None, capi.TPW_F32, 1, 2, 3, 8, s, None, None, None, 4, 0, 0, 1.0, None, s, None) == 1
    assert lib.tpw_rotary(None, capi.TPW_F32, 1, 2, 0, 8, s, None, None, None, 4, 0, 0, 1.0, None, s, None) == 0


def test_workspaces_of_empty_and_of_huge_calls():
    """Sizes that divide nothing: no heads, no batch, no rows, and counts whose product passes 64 bits.
    In a process of its own, as a trapped division would end the test run."""
    code = """
import ctypes as C
from torchpairwise_amd import _capi as capi
lib = capi.lib()
def sizes(dtype, b, h, hk, n, m, d):
    a = capi.AttentionDesc(dtype=dtype, batch=b, heads=h, key_heads=hk, n=n, m=m, d=d, dv=d, scale=1.0)
    for name, _ in a._fields_:
        if name.endswith("_strides"):
            getattr(a, name)[2] = d
    return lib.tpw_attention_workspace_size(C.byref(a)), lib.tpw_attention_backward_workspace_size(C.byref(a))
for dtype in (capi.TPW_F32, capi.TPW_BF16):
    for d in (64, 96, 128, 192, 256):
        for b, h, hk, n, m in ((1, 0, 1, 8, 8), (0, 1, 1, 8, 8), (0, 0, 2, 8, 8), (2, 0, 2, 0, 8), (2, 4, 2, 8, 0),
                               (2, 4, 2, 0, 8), (0, 4, 2, 5000, 5000)):
            forward, backward = sizes(dtype, b, h, hk, n, m, d)
            rows = b * h * n
            assert forward >= 0 and backward >= 12 * rows and (rows or forward == 0), (b, h, hk, n, m, d)
            if rows * m == 0:  # nothing to split, keep or copy
                assert backward <= 12 * rows + 12, (b, h, hk, n, m, d, backward)
        sizes(dtype, 1, 16, 1, 1 << 30, 1 << 30, d)
print("done")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).parent.parent, capture_output=True, text=True)
    assert r.returncode == 0 and "done" in r.stdout, (r.returncode, r.stdout, r.stderr[-2000:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_c_entries_without_statistics(dtype):
    """The C entry called directly, without statistics or rests, gives the operator's bits."""
    q, k, v = on("cuda", rows(2, 4, 70, 64, 1, dtype), rows(2, 2, 300, 64, 2, dtype), rows(2, 2, 300, 64, 3, dtype))
    out = torch.empty_like(q)
    a = _desc(q, k, v, out)
    ws = torch.empty(max(capi.lib().tpw_attention_workspace_size(C.byref(a)), 1), dtype=torch.uint8, device="cuda")
    capi.call("tpw_attention", C.byref(a), ws.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert_equal(out, tp.attention(q, k, v))


def test_gradients_against_differences():
    g = gen(3)
    q, k, v = (torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)
               for s in ((2, 4, 6, 5), (2, 2, 9, 5), (2, 2, 9, 3)))
    mask = torch.rand(6, 9, generator=g) < 0.6
    mask[2] = False
    bias = torch.randn(2, 1, 6, 9, generator=g, dtype=torch.float64)
    for kw in ({}, {"causal": True, "scale": -0.7}, {"mask": mask}, {"mask": bias, "lengths": torch.tensor([9, 4])}):
        assert torch.autograd.gradcheck(lambda *x: tp.attention(*x, **kw), (q, k, v)), kw
    f, s = tp.rotary_frequencies(4, scaling="parts", factor=4.0, original_length=100)
    for inter in (False, True):
        assert torch.autograd.gradcheck(
            lambda x: tp.rotary_embedding(x, torch.arange(6) * 11, f, interleaved=inter, scale=s), (q,))


@pytest.mark.parametrize("device", DEVICES)
def test_forward_mode_is_refused(device):
    """A tangent on any operand raises, with and without gradients enabled: none is dropped."""
    ops = dict(zip("qkv", on(device, rows(1, 2, 3, 8, 1), rows(1, 2, 5, 8, 2), rows(1, 2, 5, 4, 3))))
    ops["mask"] = torch.zeros(3, 5, device=device)
    for name, x in ops.items():
        for enabled in (True, False):
            with forward_ad.dual_level(), torch.set_grad_enabled(enabled):
                args = dict(ops, **{name: forward_ad.make_dual(x, torch.ones_like(x))})
                with pytest.raises(RuntimeError, match="forward-mode"):
                    tp.attention(*args.values())
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.func.jvp(lambda y: tp.attention(*dict(ops, **{name: y}).values()), (x,), (torch.ones_like(x),))
    # a dual level without tangents changes nothing
    with forward_ad.dual_level():
        assert_equal(tp.attention(*ops.values()), tp.attention(*ops.values()))


@pytest.mark.parametrize("device", DEVICES)
def test_a_graph_traced_without_gradients_gives_them(device):
    """A call recorded on operands without gradients, run on operands that require them."""
    q, k, v, grad = rows(1, 4, 9, 16, 1), rows(1, 2, 21, 16, 2), rows(1, 2, 21, 8, 3), rows(1, 4, 9, 8, 4)
    bias = randn(9, 21, seed=5)
    dq, dk, dv, dg, db = on(device, q, k, v, grad, bias)
    graph = make_fx(lambda a, b, c, m: tp.attention(a, b, c, m, causal=True))(dq, dk, dv, db)
    want = reference(q, k, v, bias, True, grad=grad)
    for which in range(3):  # each operand alone
        leaves = [x.detach().clone().requires_grad_(i == which) for i, x in enumerate((dq, dk, dv))]
        out = graph(*leaves, db)
        assert_close(out, want["out"], rtol=0.0, atol=want["tol_out"] + TINY)
        name = ("dq", "dk", "dv")[which]
        (got,) = torch.autograd.grad(out, leaves[which], dg)
        assert_close(got, want[name], rtol=0.0, atol=want["tol_" + name] + TINY, what=name)
        with torch.no_grad():
            assert not graph(*leaves, db).requires_grad
    with pytest.raises(RuntimeError, match="mask has no gradient"):
        graph(dq, dk, dv, db.clone().requires_grad_())


# ---------------------------------------------------------------- single tokens, long rows of keys
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,h,hk,m,d,dv", [(1, 1, 1, 5000, 64, 64), (1, 16, 2, 4097, 128, 128), (1, 8, 1, 3001, 256, 256),
                                          (4, 8, 2, 2050, 96, 128), (3, 40, 1, 1030, 128, 64), (1, 3, 3, 700, 50, 50),
                                          (2, 16, 1, 9000, 128, 128)])
def test_few_rows_over_many_keys(dtype, n, h, hk, m, d, dv):
    lengths = torch.tensor([m, m // 3, 1])
    check("cuda", rows(3, h, n, d, 1, dtype), rows(3, hk, m, d, 2, dtype, True), rows(3, hk, m, dv, 3, dtype),
          causal=n > 1, lengths=lengths, grad=rows(3, h, n, dv, 4, dtype) if m < 3000 else None)
    g = torch.rand(3, h, n, m, generator=gen(5)) < 0.3
    check("cuda", rows(3, h, n, d, 1, dtype), rows(3, hk, m, d, 2, dtype), rows(3, hk, m, dv, 3, dtype), g, lengths=lengths)
    bias = torch.randn(h, 1, m, generator=gen(6))
    bias[:, :, ::5] = -math.inf
    check("cuda", rows(3, h, n, d, 1, dtype), rows(3, hk, m, d, 2, dtype), rows(3, hk, m, dv, 3, dtype), bias)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,h,hk,m,d", [(1, 1, 1, 5000, 64), (1, 16, 2, 4097, 128), (1, 8, 1, 3001, 256), (4, 8, 2, 2050, 96),
                                        (3, 40, 1, 1030, 128), (1, 3, 3, 700, 50), (2, 16, 1, 9000, 128), (130, 16, 4, 2500, 64),
                                        (140, 8, 8, 2200, 128), (70, 4, 4, 300, 192)])
def test_every_key_counts_once(device, dtype, n, h, hk, m, d):
    """Equal weights and one-hot values: feature f of a row that sees L keys is the number of keys j < L with
    j % d == f over L, so that one key lost or read twice shows at any length and in any type."""
    q, k = rows(3, h, n, d, 1, dtype), rows(3, hk, m, d, 2, dtype)
    v = torch.eye(d, dtype=dtype)[torch.arange(m) % d].expand(3, hk, m, d)
    lengths = torch.tensor([m, m // 2 + 1, 65])
    seen = (lengths[:, None] - n + 1 + torch.arange(n)).clamp(min=0)[:, None, :, None]  # causal: of row i
    count = (seen - torch.arange(d) + d - 1) // d
    # the numerators, their sum and the weights of parts are whole numbers: 1 / sum, the product and the
    # result's rounding are left
    rtol = torch.finfo(dtype).eps / 2 + 8 * 2.0 ** -24
    assert count.max() * rtol < 0.5  # a key more or less is at least twice the bound
    out = tp.attention(*on(device, q, k), v.to(device), causal=True, lengths=lengths.to(device), scale=0.0)
    want = (count / seen.clamp(min=1).double()).expand(3, h, n, d)
    assert_close(out, want, rtol=rtol, atol=0.0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,h,hk,m,d", [(1, 1, 1, 5000, 64), (1, 16, 2, 4098, 128), (1, 8, 1, 3002, 256), (4, 8, 2, 2050, 96),
                                        (2, 16, 1, 9000, 128), (140, 8, 8, 2200, 128), (70, 4, 4, 300, 192),
                                        (300, 64, 64, 400, 128)])
def test_every_key_counts_once_in_the_gradients(device, dtype, n, h, hk, m, d):
    """Equal weights, one-hot keys and values of 1 and -1 in turn: the scores' gradients are 1 / m and -1 / m, so
    that feature f of dq is the number of keys j with j % d == f over m, with the sign of f.  dv of every key is
    the number of rows that see it over m."""
    q = torch.zeros(1, h, n, d, dtype=dtype)
    k = torch.eye(d, dtype=dtype)[torch.arange(m) % d].expand(1, hk, m, d).contiguous()
    sign = 1.0 - 2.0 * (torch.arange(m) % 2)
    v, grad = torch.zeros(1, hk, m, 8, dtype=dtype), torch.zeros(1, h, n, 8, dtype=dtype)
    v[..., 0], grad[..., 0] = sign.to(dtype), 1.0
    leaves = [x.requires_grad_() for x in on(device, q, k, v)]
    out = tp.attention(*leaves, scale=1.0)
    assert not out.any()
    dq, dk, dv = torch.autograd.grad(out, leaves, *on(device, grad))
    count = (m - torch.arange(d) + d - 1) // d
    # 1 / m, its rounding for the products (the gradients' type), sums of equal terms, the result's rounding
    eps = torch.finfo(dtype).eps / 2
    rtol = 2 * eps + (int(count.max()) + 8) * 2.0 ** -24
    assert count.max() * rtol < 1  # a key more or less is beyond the bound
    assert_close(dq, (count * sign[:d] / m).expand(1, h, n, d), rtol=rtol, atol=0.0, what="dq")
    assert not dk.any()
    rows_of_key = h // hk * n
    rtol = 2 * eps + (rows_of_key + 8) * 2.0 ** -24
    want = torch.zeros(1, hk, m, 8, dtype=torch.float64)
    want[..., 0] = rows_of_key / m
    assert_close(dv, want, rtol=rtol, atol=0.0, what="dv")
    if dtype == F32 or rows_of_key <= 100:
        assert rows_of_key * rtol < 1  # a row more or less is beyond the bound


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,h,hk,n,m,d,dv", [(BF16, 8, 8, 140, 2200, 128, 128), (BF16, 8, 4, 140, 3000, 128, 128),
                                                 (F32, 16, 4, 130, 2500, 64, 64), (F32, 16, 4, 133, 2500, 64, 62),
                                                 (BF16, 16, 4, 130, 2500, 64, 64), (F32, 8, 4, 140, 3000, 128, 128)])
def test_parts_of_many_rows(dtype, h, hk, n, m, d, dv):
    """9 to 32 parts of enough rows that a thread joins four features of all of them; parts without keys."""
    q, k, v = rows(1, h, n, d, 1, dtype), rows(1, hk, m, d, 2, dtype), rows(1, hk, m, dv, 3, dtype)
    if dv == d:
        a = _desc(q, k, v, torch.zeros(1, h, n, dv, dtype=dtype))
        parts = capi.lib().tpw_attention_workspace_size(C.byref(a)) / (4 * h * n * (dv + 2))
        assert 8 < parts <= 32 and parts == int(parts) and h * n * dv // 4 >= 32768
    check("cuda", q, k, v, causal=True, grad=rows(1, h, n, dv, 4, dtype))
    check("cuda", q, k, v, lengths=torch.tensor([100]))
    bias = randn(h, n, m, seed=5)
    bias[:, ::3, 40:] = -math.inf
    bias[:, 1::7] = -math.inf
    check("cuda", q, k, v, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_longer_sequences(dtype, causal, d):
    b, h, hk, n = 1, 4, 2, 700
    check("cuda", rows(b, h, n, d, 1, dtype), rows(b, hk, n, d, 2, dtype), rows(b, hk, n, d, 3, dtype), causal=causal,
          grad=rows(b, h, n, d, 4, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("d,dv", [(128, 128), (90, 72), (256, 256), (140, 256)])
@pytest.mark.parametrize("kind", ["all", "causal", "keep", "bias", "ragged"])
def test_many_heads_of_wide_rows(kind, d, dv):
    """fp32 calls that fill the GPU keep the scores' gradients for the products."""
    b, h, hk, n, m = 8, 16, 8, 170, 330
    g = gen(9)
    mask = None
    if kind == "keep":
        mask = torch.rand(n, m, generator=g) < 0.3
        mask[17] = False
    elif kind == "bias":
        mask = torch.randn(h, n, m, generator=g)
        mask[:, :, 40:90] = -math.inf
    lengths = torch.tensor([330, 0, 1, 31, 128, 129, 300, 64]) if kind == "ragged" else None
    check("cuda", rows(b, h, n, d, 1, F32, True), rows(b, hk, m, d, 2), rows(b, hk, m, dv, 3, F32, True), mask,
          causal=kind in ("causal", "ragged"), lengths=lengths, grad=rows(b, h, n, dv, 4), what=kind)


@pytest.mark.gpu
def test_heads_in_several_rounds():
    """More kept gradients than the workspace holds at a time: first and last heads of 20."""
    h, n, d = 20, 4096, 72
    q, k, v, grad = (rows(1, h, n, d, i, F32) for i in range(1, 5))
    leaves = [x.cuda().requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(tp.attention(*leaves, causal=True), leaves, grad.cuda())
    for i in (0, 19):
        want = reference(*(x[:, i:i + 1] for x in (q, k, v)), causal=True, grad=grad[:, i:i + 1])
        for name, x in zip(("dq", "dk", "dv"), got):
            assert_close(x[:, i:i + 1], want[name], rtol=0.0, atol=want["tol_" + name] + TINY, what=f"head {i} {name}")


@pytest.mark.gpu
def test_chunk_over_a_cache_equals_the_whole():
    """Queries in chunks over a growing cache with lengths give the rows of one causal call."""
    h, hk, n, d = 4, 2, 300, 64
    q, k, v = on("cuda", rows(1, h, n, d, 1, BF16), rows(1, hk, n, d, 2, BF16), rows(1, hk, n, d, 3, BF16))
    whole = tp.attention(q, k, v, causal=True).float().cpu()
    got = [tp.attention(q[:, :, a:b], k, v, causal=True, lengths=torch.tensor([b], device="cuda"))
           for a, b in ((0, 1), (1, 130), (130, 131), (131, 300))]
    bound = reference(*(x.cpu() for x in (q, k, v)), causal=True)["tol_out"]
    assert_close(torch.cat(got, 2), whole, rtol=0.0, atol=2 * bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_repeats_and_other_streams(dtype):
    """The same call gives the same bits, on another stream too."""
    args = on("cuda", rows(2, 8, 200, 128, 1, dtype), rows(2, 2, 333, 128, 2, dtype), rows(2, 2, 333, 128, 3, dtype))
    grad = rows(2, 8, 200, 128, 4, dtype).cuda()
    leaves = [x.requires_grad_() for x in args]

    def call():
        out = tp.attention(*leaves, causal=True)
        return out, *torch.autograd.grad(out, leaves, grad)

    first = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(2):
        with torch.cuda.stream(side):
            again = call()
        side.synchronize()
        for a, b in zip(first, again):
            assert_equal(a, b)


@pytest.mark.gpu
def test_replays_of_a_graph():
    q, k, v = on("cuda", rows(2, 8, 1, 128, 1, BF16), rows(2, 2, 1500, 128, 2, BF16), rows(2, 2, 1500, 128, 3, BF16))
    lengths = torch.tensor([700, 1500], device="cuda")
    f, _ = tp.rotary_frequencies(128, device="cuda")
    pos = torch.tensor([[699], [1499]], device="cuda")

    def call():
        return tp.attention(tp.rotary_embedding(q, pos, f), k, v, lengths=lengths)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        q.add_(0.25)
        lengths[0] = 100 * i
        graph.replay()
        torch.cuda.synchronize()
        assert_equal(out, call(), f"replay {i}")
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Keys and values whose rows lie 6 GiB apart in all, in one head."""
    m, d, stride = 800, 64, 1 << 22  # 8 MiB between rows
    k, v = rows(1, 1, m, d, 2, BF16), rows(1, 1, m, d, 3, BF16)
    buf = torch.zeros(m * stride, dtype=BF16, device="cuda")
    view = buf.view(1, 1, m, stride)
    view[..., :d] = k.cuda()
    view[..., d:2 * d] = v.cuda()
    for n in (1, 70):
        q, grad = rows(1, 1, n, d, 1, BF16), rows(1, 1, n, d, 4, BF16)
        want = reference(q, k, v, grad=grad)
        dq = q.cuda().requires_grad_()
        out = tp.attention(dq, view[..., :d], view[..., d:2 * d])
        assert_close(out, want["out"], rtol=0.0, atol=want["tol_out"])
        (g,) = torch.autograd.grad(out, dq, grad.cuda())
        assert_close(g, want["dq"], rtol=0.0, atol=want["tol_dq"])


@pytest.mark.gpu
def test_neighbour_mask_feeds_attention():
    """Attention over a neighbour graph of the framework's own masks; isolated points give zeros."""
    x = randn(300, 32, seed=1).cuda()
    x[7] += 1000.0
    mask = tp.radius_neighbors_mask(x, epsilon=6.0)
    if mask.shape == (300, 300):
        mask = mask & ~torch.eye(300, dtype=torch.bool, device="cuda")
    want = reference(*(x.cpu()[None, None],) * 3, mask.cpu(), scale=0.05)
    out = tp.attention(x, x, x, mask, scale=0.05)
    assert not out[7].any()
    assert_close(out, want["out"][0, 0], rtol=0.0, atol=want["tol_out"][0, 0] + TINY)


@pytest.mark.parametrize("device", DEVICES)
def test_example(device):
    """The example's parts together: training lowers the loss, tokens over a cache give what one call
    gives, neighbours correct labels."""
    import importlib.util
    from pathlib import Path

    spec = importlib.util.spec_from_file_location("example", Path(__file__).parent.parent / "examples" / "attention.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    r = example.main(device, steps=60)
    assert r["last_loss"] < 0.5 * r["first_loss"]
    assert r["decode_gap"] < 1e-3  # logits of order 10 in fp32
    assert r["labels_after"] > r["labels_before"]


# ---------------------------------------------------------------- rotary
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,h,n,d,width,rf", [(1, 1, 1, 2, 2, False), (2, 3, 5, 64, 64, True), (16, 8, 1, 128, 128, False),
                                             (3, 5, 103, 118, 50, True), (1, 2, 33, 96, 32, False), (2, 2, 7, 9, 6, False),
                                             (1, 4, 300, 256, 128, True), (2, 2, 4, 20, 0, False)])
def test_rotary(device, dtype, interleaved, b, h, n, d, width, rf):
    x, grad = rows(b, h, n, d, 1, dtype, rf), rows(b, h, n, d, 2, dtype, rf)
    f = 10000.0 ** (-torch.arange(width // 2, dtype=torch.float64) / max(width // 2, 1))
    pos = torch.randint(0, 1 << 20, (b, n), generator=gen(3))
    dx, dg = on(device, x, grad)
    dx.requires_grad_()
    # cos, sin (2 u each), two products and a sum in fp32, the result's rounding
    b_round = torch.finfo(dtype).eps / 2
    for p, scale in ((pos, 1.0), (pos[:1], 1.3), (pos[0], 1.0)):
        y = tp.rotary_embedding(dx, p.to(device), f.to(device), interleaved=interleaved, scale=scale)
        assert y.shape == x.shape and y.dtype == dtype
        want = rotate(x, p, f, interleaved, scale)
        size = rotate(x.abs(), torch.zeros_like(p), f, interleaved, scale)
        pair = _partner(x.abs().double(), width, interleaved, scale)
        assert_close(y, want, rtol=b_round, atol=8 * 2.0 ** -24 * (size + pair), what="rotary")
        assert_equal(y[..., width:], x[..., width:], "features past the width")
        (g,) = torch.autograd.grad(y, dx, dg)
        want = rotate(grad, p, f, interleaved, scale, inverse=True)
        size = rotate(grad.abs(), torch.zeros_like(p), f, interleaved, scale)
        pair = _partner(grad.abs().double(), width, interleaved, scale)
        assert_close(g, want, rtol=b_round, atol=8 * 2.0 ** -24 * (size + pair), what="rotary gradient")


def _partner(x, width, interleaved, scale):
    """Each rotated feature's partner, times scale."""
    r = x[..., :width]
    if interleaved:
        y = r.unflatten(-1, (width // 2, 2)).flip(-1).flatten(-2)
    else:
        y = r.roll(width // 2, -1) if width else r
    return torch.cat([y * scale, torch.zeros_like(x[..., width:])], -1)


@pytest.mark.parametrize("device", DEVICES)
def test_rotary_strides(device):
    f = torch.rand(8, dtype=torch.float64, generator=gen(1))
    base = randn(2, 3, 11, 45, seed=2)
    pos = torch.arange(22).view(1, 22)[:, ::2]
    for x in (base[..., 1:33], base[..., 5:37:2], base[:, :, ::2, :17][:, :, :, 1:], base.mT[:, :, :16, :11].mT):
        want = rotate(x, pos[:, :x.shape[2]], f)
        got = tp.rotary_embedding(on(device, x)[0], pos.to(device)[:, :x.shape[2]], f.to(device))
        assert_close(got, want, rtol=2.0 ** -22, atol=2.0 ** -20)
    y = tp.rotary_embedding(on(device, randn(11, 16, seed=3))[0], pos[0].to(device).int(), f.float().to(device))
    assert_close(y, rotate(randn(11, 16, seed=3)[None, None], pos, f.float())[0, 0], rtol=2.0 ** -22, atol=2.0 ** -20)


def test_rotary_makes_products_depend_on_the_distance():
    f, _ = tp.rotary_frequencies(32)
    q, k = randn(1, 32, seed=1).double(), randn(1, 32, seed=2).double()
    at = [(tp.rotary_embedding(q, torch.tensor([a]), f) @ tp.rotary_embedding(k, torch.tensor([a + 5]), f).T).item()
          for a in (0, 17, 100000)]
    assert max(at) - min(at) < 1e-9


def test_rotary_frequencies():
    f, s = tp.rotary_frequencies(8)
    assert f.dtype == torch.float64 and s == 1.0
    assert_close(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14, atol=0.0)
    lin, s = tp.rotary_frequencies(8, scaling="linear", factor=4.0)
    assert_close(lin, f / 4, rtol=1e-14, atol=0.0)
    b, s = tp.rotary_frequencies(8, scaling="base", factor=4.0)
    assert abs(b[0] - 1) < 1e-14 and abs(b[-1] / f[-1] - 0.25) < 1e-12 and s == 1.0
    p, s = tp.rotary_frequencies(64, scaling="parts", factor=8.0, original_length=4096)
    f = tp.rotary_frequencies(64)[0]
    turns = 4096 * f / (2 * math.pi)
    assert_close(p[turns > 40], f[turns > 40], rtol=1e-14, atol=0.0)
    assert_close(p[turns < 0.8], f[turns < 0.8] / 8, rtol=1e-14, atol=0.0)
    assert ((p <= f) & (p >= f / 8 * (1 - 1e-14))).all() and abs(s - (0.1 * math.log(8.0) + 1)) < 1e-15
    for bad in ({"width": 7}, {"width": 8, "base": 1.0}, {"width": 8, "scaling": "x"}, {"width": 8, "factor": 2.0},
                {"width": 8, "scaling": "linear", "factor": 0.5}, {"width": 8, "scaling": "parts", "factor": 2.0},
                {"width": 8, "scaling": "parts", "factor": 2.0, "original_length": 64, "fast": 1.0}):
        with pytest.raises(ValueError):
            tp.rotary_frequencies(**bad)


@pytest.mark.parametrize("width,base,length,factor", [(128, 1e4, 131072, 4.0), (64, 1e4, 1 << 20, 4.0), (128, 1e4, 65536, 8.0),
                                                      (64, 1e4, 4096, 2.0), (32, 500.0, 100, 4.0), (16, 1e4, 4, 4.0),
                                                      (2, 1e4, 100, 4.0)])
def test_parts_of_the_frequencies_by_their_turns(width, base, length, factor):
    """Kept where a pair makes 32 turns or more over the original length, divided by the factor where it makes
    one or fewer, a line over the pairs between, also where its ends lie outside the pairs there are."""
    f = tp.rotary_frequencies(width, base)[0]
    got = tp.rotary_frequencies(width, base, scaling="parts", factor=factor, original_length=length)[0] / f
    turns = length * f / (2 * math.pi)
    assert_close(got[turns >= 32.0], torch.ones_like(got[turns >= 32.0]), rtol=1e-12, atol=0.0)
    assert_close(got[turns <= 1.0], torch.full_like(got[turns <= 1.0], 1 / factor), rtol=1e-12, atol=0.0)
    # turns fall by `step` in their logarithm from pair to pair: where they reach 32 and 1
    step = 2 * math.log(base) / width
    ends = [math.log(length / (2 * math.pi * t)) / step for t in (32.0, 1.0)]
    first, last = math.floor(ends[0]), math.ceil(ends[1])
    share = ((torch.arange(width // 2, dtype=torch.float64) - first) / (last - first)).clamp(0.0, 1.0)
    assert_close(got, 1.0 - share * (1.0 - 1 / factor), rtol=1e-12, atol=0.0)


@pytest.mark.parametrize("device", DEVICES)
def test_frequencies_held_as_a_parameter(device):
    """They have no gradient, so they are refused only where one would be lost."""
    x, pos = randn(2, 3, 5, 16, seed=1).to(device), torch.arange(5, device=device)
    f = torch.rand(8, dtype=torch.float64, generator=gen(2)).to(device)
    held = torch.nn.Parameter(f)
    with torch.no_grad():
        assert_equal(tp.rotary_embedding(x, pos, held), tp.rotary_embedding(x, pos, f))
    with torch.inference_mode():
        assert_equal(tp.rotary_embedding(x, pos, held), tp.rotary_embedding(x, pos, f))
    leaf = x.clone().requires_grad_()
    assert tp.rotary_embedding(leaf, pos, held.detach()).requires_grad
    for y in (x, leaf):
        with pytest.raises(RuntimeError, match="frequencies have no gradient"):
            tp.rotary_embedding(y, pos, held)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("enabled", [True, False])
def test_rotary_refuses_tangents(device, enabled):
    x, f = randn(2, 3, 5, 16, seed=1).to(device), torch.rand(8, dtype=torch.float64, generator=gen(2)).to(device)
    pos = torch.arange(5, device=device)
    with forward_ad.dual_level(), torch.set_grad_enabled(enabled):
        for args in ((forward_ad.make_dual(x, x), pos, f), (x, pos, forward_ad.make_dual(f, f))):
            with pytest.raises(RuntimeError):
                tp.rotary_embedding(*args)

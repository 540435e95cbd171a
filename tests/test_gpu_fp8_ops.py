"""Codes and products in 8-bit floating point with a scale for each block of 128, on the GPU, against numpy in 64 bits
(fp8_reference.py).  Codes and powers of two are compared bit by bit; tolerances follow from the operations' roundings and
stand beside each comparison."""
import math

import numpy as np
import pytest

import fp8_reference as R
import pyPhantom as ph
from test_gpu_clear_ops import TYPES, dtype_of, f64, layouts, normal

pytestmark = pytest.mark.gpu

U = R.U
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # half a step, relative
WIDTHS = [1, 2, 7, 8, 9, 63, 100, 127, 128, 129, 200, 255, 256, 500, 1000, 1024, 2050, 4096, 5119, 8192, 16384, 20003, 24576, 40001,
          40960]


def numbers(codes):
    return codes.float().cpu().double().numpy()


def check_quantized(codes, scales, x, rows=1):
    """Every code and scale: the scale is a power of two, the quotient by it exact, the rounding the definition's."""
    want, steps = R.quantized(f64(x), rows)
    assert codes.shape == x.shape and str(codes.dtype) == "torch.float8_e4m3fn"
    assert np.array_equal(f64(scales), steps, equal_nan=True)
    assert np.array_equal(numbers(codes), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_quantize_rows(dev, dtype, width):
    for rows in (1, 3, 37):
        x = normal(width + rows, rows, width, dtype=dtype, dev=dev)
        for kind in ("dense", "apart", "odd"):
            codes, scales = ph.quantize_fp8(layouts(x, kind))
            assert scales.shape == (rows, R.spans(width)) and (rows == 1 or scales.stride(0) == 1)
            check_quantized(codes, scales, x)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 128), (5, 7), (127, 129), (128, 128), (129, 1000), (300, 257), (1000, 64)])
def test_quantize_squares(dev, dtype, rows, width):
    x = normal(rows * width, rows, width, dtype=dtype, dev=dev)
    for kind in ("dense", "apart", "odd"):
        codes, scales = ph.quantize_fp8(layouts(x, kind), 128)
        assert scales.shape == (R.spans(rows), R.spans(width)) and scales.is_contiguous()
        check_quantized(codes, scales, x, 128)


def test_quantize_edges(dev):
    """Zeros, the border between two powers, subnormal and the largest numbers, ties, NaN and infinities; blocks beside
    them are not touched."""
    import torch

    inf, nan = math.inf, math.nan
    rows = [[0.0, -0.0], [448.0, 1.0], [448.00003, 1.0], [447.99997, 1.0], [1e-45, -1e-45], [2.0 ** -126, 3e-39],
            [3.4028235e38, -1e38], [nan, 1], [1, inf], [-inf, nan], [2.0 ** -118 * 1.75, 1e-37], [2.0 ** -118 * 1.76, 1e-37]]
    x = torch.zeros((len(rows), 300), device=dev)
    x[:, 130:132] = torch.tensor(rows, device=dev)
    x[:, 140] = 0.0
    x[:, 3] = 5.0
    # every tie between two codes, and its neighbours
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    codes = codes[codes.isfinite()].unique()
    ties = ((codes[1:] + codes[:-1]) / 2).to(dev)
    ties = torch.cat([ties, torch.nextafter(ties, torch.full_like(ties, inf)), torch.nextafter(ties, torch.full_like(ties, -inf))])
    y = torch.zeros((ties.numel(), 128), device=dev)
    y[:, 7], y[:, 100] = ties, 448.0
    for v in (x, y):
        for rows_of in (1, 128):
            c, s = ph.quantize_fp8(v, rows_of)
            check_quantized(c, s, v, rows_of)
    c, s = ph.quantize_fp8(x)
    assert torch.isnan(s[7:10, 1]).all() and (c[7:10, 128:256].float() == 0).all() and (s[7:10, 0] > 0).all()


@pytest.mark.parametrize("shape", [(0, 5), (5, 0), (0, 0), (2, 0, 9), (2, 3, 130), (130,)])
def test_quantize_shapes(dev, shape):
    import torch

    x = torch.randn(shape, device=dev)
    codes, scales = ph.quantize_fp8(x)
    assert codes.shape == x.shape and scales.shape == (*shape[:-1], R.spans(shape[-1]))
    if x.numel():
        check_quantized(codes.reshape(-1, shape[-1]), scales.reshape(-1, scales.shape[-1]), x.reshape(-1, shape[-1]))
    if len(shape) == 2:
        codes, scales = ph.quantize_fp8(x, 128)
        assert scales.shape == (R.spans(shape[0]), R.spans(shape[1]))


def test_quantize_many_rows(dev):
    """More workgroups than one dimension of the grid holds, and bytes past 2^32."""
    import torch

    x = torch.zeros((1 << 21, 1040), dtype=torch.bfloat16, device=dev)
    x[-1, -1], x[0, 0], x[1 << 20, 129] = 3.0, -7.0, 448.0
    codes, scales = ph.quantize_fp8(x)
    assert codes[-1, -1].float() * scales[-1, -1] == 3 and codes[0, 0].float() * scales[0, 0] == -7
    assert codes[1 << 20, 129].float() == 448 and scales[1 << 20, 1] == 1
    assert int((scales != 0).sum()) == 3


# ------------------------------------------------------------- norm
def check_norm(codes, scales, x, w, eps, r, terms):
    """y = x + r and y w have one rounding each, so a value is off by 2 U and a block's largest too: the power of two is the
    definition's unless that largest is within 4 U of the border, and a code is within half a step (and 4 U of its
    value).  The factor has the sum's roundings (halved by the root) and 4 of its own."""
    y = f64(x) if r is None else f64(x) + f64(r)
    factor = 1 / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
    v = y * f64(w)
    s = f64(scales)
    power = np.exp2(np.rint(np.log2(np.maximum(s, 1e-300) / factor)))
    tops = R.block_tops(v)
    some = s > 0
    assert np.array_equal(some, tops > 0)
    assert np.all(np.abs(s / factor - power)[some] <= ((8 + terms / 2) * U * power)[some])
    assert np.all((power * 448 >= tops * (1 - 4 * U))[some]) and np.all((power * 224 <= tops * (1 + 4 * U))[some])
    q = np.where(R.spread(some, v.shape), v / R.spread(power, v.shape), 0.0)
    c = numbers(codes)
    # the distance of codes around q; past a power of two it doubles, and q may be the one below
    assert np.all(np.abs(c - q) <= R.e4m3_step(q * (1 + 4 * U)) / 2 + 4 * U * np.abs(q))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_norm(dev, dtype, width):
    import torch

    for rows in (1, 3, 37):
        x, r = (normal(width + rows + k, rows, width, dtype=dtype, dev=dev) for k in (0, 50000))
        w = normal(width, width, dtype=dtype, dev=dev, spread=0.3)
        for kind in ("dense", "odd"):
            for res in (None, r):
                args = layouts(x, kind), layouts(w, kind), 1e-5, None if res is None else layouts(res, kind)
                codes, scales, total = ph.rms_norm_fp8(*args)
                check_norm(codes, scales, x, w, 1e-5, res, width / 64 + 20)
                if res is None:
                    assert total is args[0]
                else:  # one rounding to 32 bits, one to the type: what torch does
                    assert torch.equal(total, (x.float() + r.float()).to(x.dtype))


def test_norm_edges(dev):
    import torch

    inf, nan = math.inf, math.nan
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.ones((9, 300), device=dev, dtype=dtype)
        r = torch.ones_like(x)
        w = torch.ones(300, device=dev, dtype=dtype)
        x[0], r[0] = 0, 0       # a row of zeros: eps keeps the norm finite
        x[1], r[1] = 5, -5      # the residual takes everything away
        x[2, 17] = nan
        x[3, 299] = inf
        r[4, 0], x[4, 0] = -inf, inf
        x[5], r[5] = 1e30, 0    # squares pass 32 bits
        x[6, 128:256], r[6, 128:256] = 0, 0  # one block of zeros
        codes, scales, total = ph.rms_norm_fp8(x, w, 1e-6, r)
        assert (codes[:2].float() == 0).all() and (scales[:2] == 0).all() and (total[:2] == 0).all()
        assert torch.isnan(scales[2:6]).all() and (codes[2:6].float() == 0).all()
        assert (scales[6, 1] == 0) and (codes[6, 128:256].float() == 0).all() and (scales[6, [0, 2]] > 0).all()
        check_norm(codes[6:], scales[6:], x[6:], w, 1e-6, r[6:], 30)
        # a weight that is not finite: its block alone, unless y is 0 in it
        w2 = w.clone()
        w2[130] = inf
        codes, scales, _ = ph.rms_norm_fp8(x[7:], w2, 1e-6)
        assert torch.isnan(scales[:, 1]).all() and torch.isfinite(scales[:, [0, 2]]).all()
        assert (codes[:, 128:256].float() == 0).all()
        codes, scales, _ = ph.rms_norm_fp8(x[:1] * 0, w, 0.0)  # nothing at all, not even eps
        assert (scales == 0).all() and (codes.float() == 0).all()


@pytest.mark.parametrize("size", [1e-24, 1e-30, 1e-38, 1e-42])
@pytest.mark.parametrize("width", [100, 3000, 40001])
def test_norm_small_squares(dev, size, width):
    """Squares that vanish in 32 bits: the norm is the values' all the same.  Subnormal values are their own rounding."""
    import torch

    x = (torch.randn((2, width), generator=torch.Generator().manual_seed(width)) * size).to(dev)
    w = torch.ones(width, device=dev)
    codes, scales, _ = ph.rms_norm_fp8(x, w, 0.0)
    y = f64(x)
    factor = 1 / np.sqrt((y * y).mean(-1, keepdims=True))
    want = R.power_for(R.block_tops(y)) * factor
    assert np.all(np.abs(f64(scales) - want) <= (12 + width / 512) * U * want)
    assert np.array_equal(numbers(codes), R.quantized(y)[0])


# ------------------------------------------------------------- products
def operands(seed, m, n, k, dev, kind="dense", wide=False):
    """(a, its scales, b, its scales) of random codes: every finite code where wide, else those of normal values."""
    import torch

    g = torch.Generator().manual_seed(seed)

    def codes(rows):
        if wide:
            c = torch.randint(0, 256, (rows, k), generator=g, dtype=torch.uint8)
            c[(c & 127) == 127] = 0
            c = c.view(torch.float8_e4m3fn)
        else:
            c = (torch.randn((rows, k), generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        c = c.to(dev)
        if kind == "dense":
            return c
        pad, off = (5, 1) if kind == "odd" else (256, 128)
        big = torch.full((rows, k + pad), 127, dtype=torch.uint8, device=dev)  # NaN codes around the rows
        big[:, off:off + k] = c.view(torch.uint8)
        return big.view(torch.float8_e4m3fn)[:, off:off + k]

    sa = torch.exp(torch.randn((m, R.spans(k)), generator=g)).to(dev)
    sb = (torch.randn((R.spans(n), R.spans(k)), generator=g) / max(k, 1) ** 0.5).to(dev)
    if kind != "odd":
        sa = sa.t().contiguous().t()
    else:
        sb = sb.t().contiguous().t()
    return codes(m), sa, codes(n), sb


def check_matmul(out, a, sa, b, sb, bias, dtype):
    """A sum of n numbers in 32 bits, in any order, is off by n U times their magnitudes (each addition by one rounding; the
    matrix unit's may cut instead, twice that); a block adds 128 products, then one for each block, each part of K and
    the bias, and a block's scale is rounded twice.  For 16-bit outputs the matrix unit also cuts, of each eight
    products, what is below 2^-13 of their largest; then the rounding to the output's type."""
    want, size, eights = R.matmul(numbers(a), f64(sa), numbers(b), f64(sb), None if bias is None else f64(bias))
    got = f64(out)
    assert got.shape == want.shape
    blocks = sa.shape[1]
    size = size + (0 if bias is None else np.abs(f64(bias)))
    room = 2 * (128 + blocks + 12) * U * size + HALF[dtype] * np.abs(want)
    if dtype != "float32":
        room += 8 * 2.0 ** -13 * eights + (2.0 ** -25 if dtype == "float16" else 0)
    with np.errstate(invalid="ignore"):
        bad = ~(np.abs(got - want) <= room)
    # from 65520 on the nearest of float16 is infinity
    over = np.isinf(got) & (got * want > 0) & (np.abs(want) + room >= 65520) & (dtype == "float16")
    bad &= ~over
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5].tolist())


SIZES = [(1, 1, 1), (1, 16, 128), (2, 17, 127), (16, 130, 129), (17, 16, 64), (5, 300, 1000), (33, 129, 4096), (100, 200, 300),
         (16, 1024, 4097), (257, 513, 256), (130, 257, 1152), (64, 64, 2048), (300, 100, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul(dev, dtype, m, n, k):
    import torch

    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dev)
    for kind in ("dense", "apart", "odd"):
        args = operands(m + n + k, m, n, k, dev, kind, wide=kind != "dense")
        for more in (None, bias):
            check_matmul(ph.fp8_matmul(*args, more, dtype_of(dtype)), *args, more, dtype)


@pytest.mark.parametrize("m,n,k", SIZES)
def test_matmul_of_float16_size(dev, m, n, k):
    """Products that float16 holds."""
    import torch

    for kind in ("dense", "odd"):
        a, sa, b, sb = operands(m + n + k, m, n, k, dev, kind)
        sa = sa * 2.0 ** -14
        out = ph.fp8_matmul(a, sa, b, sb, None, torch.float16)
        assert torch.isfinite(out).all()
        check_matmul(out, a, sa, b, sb, None, "float16")


def test_matmul_layouts_agree(dev):
    """The same numbers in other memory give the same bits."""
    import torch

    for m, n, k in ((3, 500, 1000), (200, 300, 640), (150, 1000, 1111)):
        a, sa, b, sb = operands(m, m, n, k, dev)
        for dtype in (torch.bfloat16, torch.float32):
            want = ph.fp8_matmul(a, sa, b, sb, None, dtype)
            for kind in ("apart", "odd"):
                def moved(c):
                    pad, off = (5, 1) if kind == "odd" else (256, 128)
                    big = torch.full((c.shape[0], k + pad), 255, dtype=torch.uint8, device=dev)
                    big[:, off:off + k] = c.view(torch.uint8)
                    return big.view(torch.float8_e4m3fn)[:, off:off + k]
                assert torch.equal(ph.fp8_matmul(moved(a), sa.contiguous(), moved(b), sb.t().contiguous().t(), None, dtype), want)


def test_matmul_empty(dev):
    import torch

    e = torch.float8_e4m3fn
    bias = torch.randn(6, device=dev)
    a = torch.zeros((4, 0), device=dev).to(e)
    b = torch.zeros((6, 0), device=dev).to(e)
    out = ph.fp8_matmul(a, torch.zeros((4, 0), device=dev), b, torch.zeros((1, 0), device=dev), bias, torch.float32)
    assert torch.equal(out, bias.expand(4, 6))
    a, sa, b, sb = operands(1, 2, 6, 130, dev)
    assert ph.fp8_matmul(a[:0], sa[:0], b, sb).shape == (0, 6)
    assert ph.fp8_matmul(a, sa, b[:0], sb[:0]).shape == (2, 0)


def test_matmul_leading_dimensions(dev):
    import torch

    x = torch.randn((2, 3, 200), device=dev)
    a, sa = ph.quantize_fp8(x)
    b, sb = ph.quantize_fp8(torch.randn((50, 200), device=dev), 128)
    out = ph.fp8_matmul(a, sa, b, sb, None, torch.float32)
    flat = ph.fp8_matmul(a.reshape(6, 200), sa.reshape(6, 2), b, sb, None, torch.float32)
    assert out.shape == (2, 3, 50) and torch.equal(out.reshape(6, 50), flat)
    one = ph.fp8_matmul(a[0, 0], sa[0, 0], b, sb, None, torch.float32)
    assert one.shape == (50,) and torch.allclose(one, flat[0], rtol=1e-5, atol=1e-5)


def test_matmul_nan_and_infinite_scales(dev):
    """A NaN code or scale reaches the outputs of its row, or of its 128 columns, and no others."""
    import torch

    for m, n, k in ((5, 300, 500), (200, 300, 500)):
        for dtype in (torch.bfloat16, torch.float32):
            a, sa, b, sb = operands(m, m, n, k, dev)
            clean = ph.fp8_matmul(a, sa, b, sb, None, dtype)
            sa2, sb2 = sa.clone(), sb.clone()
            sa2[3, 1], sb2[1, 2] = math.nan, math.inf
            out = ph.fp8_matmul(a, sa2, b, sb2, None, dtype)
            assert torch.isnan(out[3]).all() and not torch.isfinite(out[:, 128:256]).any()
            keep = torch.ones(m, dtype=torch.bool)
            keep[3] = False
            assert torch.equal(out[keep][:, :128], clean[keep][:, :128]) and torch.equal(out[keep][:, 256:], clean[keep][:, 256:])
            a2 = a.clone()
            a2.view(torch.uint8)[1, k - 1] = 0xff
            out = ph.fp8_matmul(a2, sa, b, sb, None, dtype)
            assert torch.isnan(out[1]).all() and torch.equal(out[2:], clean[2:])


def test_wide_outputs_count_every_product(dev):
    """One large product and small ones beside it: a 32-bit output holds them all."""
    import torch

    a = torch.zeros((3, 256), device=dev)
    a[:, :8] = torch.tensor([448.0, *([2.0 ** -9] * 7)], device=dev)
    b = torch.ones((130, 256), device=dev)
    one = torch.ones((3, 2), device=dev), torch.ones((2, 2), device=dev)
    e = torch.float8_e4m3fn
    out = ph.fp8_matmul(a.to(e), one[0], b.to(e), one[1], None, torch.float32)
    assert (out == 448 + 7 * 2.0 ** -9).all()

"""Products whose rows, or whose rows of scales, are too far apart for the tiles' 32-bit offsets (8 MiB of codes, 2^20 and
2^23 scales), and ones that just fit, against the definition in 64 bits: every type of output, sums short and long."""
import pytest

import fp8_reference as R
import pfa_native as P
import pyPhantom as ph
from test_gpu_clear_ops import TYPES, dtype_of
from test_gpu_fp8_ops import operands
from test_gpu_fp8_shapes import check_large

pytestmark = pytest.mark.gpu

FAR = 1 << 23


def spaced(t, pitch, before=0):
    """t [rows, n] with its rows `pitch` elements apart, what is between them NaN."""
    import torch

    codes = t.element_size() == 1
    v = t.view(torch.uint8) if codes else t
    rows, n = t.shape
    big = torch.full(((rows - 1) * pitch + n + before,), 127 if codes else float("nan"), dtype=v.dtype, device=t.device)
    big = big[before:].as_strided((rows, n), (pitch, 1))
    big.copy_(v)
    return big.view(t.dtype) if codes else big


def outputs_fit(sa, dtype):
    return sa * 2.0 ** -14 if dtype == "float16" else sa


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(5, 20, 300), (1, 33, 4097), (5, 20, 8200), (37, 9, 4224), (3, 300, 5000)])
def test_rows_far_apart(dev, dtype, m, n, k):
    """Blocks four at a time and one by one, a rows' end, several workgroups down and across; a bias."""
    import torch

    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dev)
    a, sa, b, sb = operands(m + n + k, m, n, k, dev)
    sa = outputs_fit(sa, dtype)
    which = [(spaced(a, FAR + 1, 3), b)] if m > 1 else []
    if n <= 40:
        which += [(a, spaced(b, FAR + 128)), (spaced(a, FAR + 128), spaced(b, FAR + 1, 1))]
    for p, q in which:
        for more in (None, bias):
            check_large(ph.fp8_matmul(p, sa, q, sb, more, dtype_of(dtype)), p, sa, q, sb, more, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [300, 4097])
def test_scales_far_apart(dev, dtype, k):
    """Rows of a's scales more than 2^20 numbers apart, rows of b's more than 2^23."""
    m, n = 18, 300
    a, sa, b, sb = operands(k, m, n, k, dev)
    sa = outputs_fit(sa, dtype)
    wide_a, wide_b = spaced(sa, (1 << 20) + 1), spaced(sb, FAR + 1)
    for p, q in ((wide_a, sb), (sa, wide_b), (wide_a, wide_b)):
        check_large(ph.fp8_matmul(a, p, b, q, None, dtype_of(dtype)), a, sa, b, sb, None, dtype)


# [M, N, K]: tiles of 256 rows, and of 256 columns, for 32-bit and 16-bit outputs
TALL = {"float32": (641, 10844, 130), "bfloat16": (385, 27687, 256), "float16": (385, 27687, 256)}
BROAD = {"float32": (8986, 642, 2048), "bfloat16": (8939, 1319, 384), "float16": (8939, 1319, 384)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows_of", ["a", "b"])
def test_rows_as_far_as_tiles_reach(dev, dtype, rows_of):
    """256 rows of a tile exactly 2^23 bytes apart, their scales 2^20 (of b 2^23) numbers: the largest offsets that are
    still a tile's."""
    m, n, k = (TALL if rows_of == "a" else BROAD)[dtype]
    assert P.fp8_plan(m, n, k, TYPES.index(dtype))[0 if rows_of == "a" else 1] == 256
    a, sa, b, sb = operands(m, m, n, k, dev)
    sa = outputs_fit(sa, dtype)
    if rows_of == "a":
        p, q, s, z = spaced(a, FAR), b, spaced(sa, 1 << 20), sb
    else:
        p, q, s, z = a, spaced(b, FAR), sa, spaced(sb, FAR)
    check_large(ph.fp8_matmul(p, s, q, z, None, dtype_of(dtype)), a, sa, b, sb, None, dtype)

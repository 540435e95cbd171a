"""Every shape of tile and every split that fp8_matmul plans with, against the definition in 64 bits."""
import pytest

import fp8_reference as R
import pyPhantom as ph
from fp8_shapes import FEW, NARROW, WIDE
from test_gpu_clear_ops import dtype_of
from test_gpu_fp8_ops import HALF, operands

pytestmark = pytest.mark.gpu


def check_large(out, a, sa, b, sb, bias, dtype):
    """As check_matmul, on the GPU; the largest product of eight is at most the product of the largest codes."""
    import torch

    (m, k), n = a.shape, b.shape[0]
    blocks = R.spans(k)

    def real(c, s, rows):
        v = torch.zeros((c.shape[0], blocks * 128), dtype=torch.float64, device=c.device)
        v[:, :k] = c.float().double()
        s = s.double().repeat_interleave(rows, 0)[:c.shape[0]].repeat_interleave(128, 1)
        eights = (v.abs().clamp_min(2.0 ** -6) * s.abs()).view(c.shape[0], -1, 8).amax(-1)
        return v * s, eights

    A, A8 = real(a, sa, 1)
    B, B8 = real(b, sb, 128)
    want = torch.mm(A, B.t().contiguous())
    size = torch.mm(A.abs(), B.abs().t().contiguous())
    if bias is not None:
        want += bias.double()
        size += bias.double().abs()
    room = 2 * (128 + blocks + 12) * R.U * size + HALF[dtype] * want.abs()
    if dtype != "float32":
        room += 8 * 2.0 ** -13 * torch.mm(A8, B8.t().contiguous()) + (2.0 ** -25 if dtype == "float16" else 0)
    far = (out.double() - want).abs()
    assert out.shape == (m, n) and torch.isfinite(out).all()
    assert bool((far <= room).all()), (float((far / room).max()), torch.nonzero(far > room)[:4].tolist())


@pytest.mark.parametrize("m,n,k", WIDE + FEW)
def test_wide(dev, m, n, k):
    import torch

    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dev)
    for kind in ("dense", "odd"):
        args = operands(m + n + k, m, n, k, dev, kind)
        check_large(ph.fp8_matmul(*args, bias, torch.float32), *args, bias, "float32")


@pytest.mark.parametrize("m,n,k", NARROW + FEW)
def test_narrow(dev, m, n, k):
    import torch

    bias = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dev)
    for kind, dtype in (("dense", "bfloat16"), ("odd", "float16")):
        a, sa, b, sb = operands(m + n + k, m, n, k, dev, kind)
        sa = sa * 2.0 ** -14  # float16 holds the outputs
        check_large(ph.fp8_matmul(a, sa, b, sb, bias, dtype_of(dtype)), a, sa, b, sb, bias, dtype)


def test_rows_far_apart(dev):
    """Rows more than 8 MiB apart are beyond the tiles' offsets, and formed all the same."""
    import torch

    n, k, pitch = 70, 300, (1 << 23) + 128
    a, sa, b, sb = operands(3, 40, n, k, dev)
    want = ph.fp8_matmul(a, sa, b, sb, None, torch.float32)

    def apart(c):
        big = torch.empty(((c.shape[0] - 1) * pitch + k,), dtype=torch.uint8, device=dev)
        v = big.as_strided((c.shape[0], k), (pitch, 1))
        v.copy_(c.view(torch.uint8))
        return v.view(torch.float8_e4m3fn)

    for out in (ph.fp8_matmul(apart(a), sa, b, sb, None, torch.float32), ph.fp8_matmul(a, sa, apart(b), sb, None, torch.float32)):
        assert torch.allclose(out, want, rtol=1e-4, atol=float(want.abs().max()) * 1e-6)
    one = a[:1].expand(40, k)  # one row over and over
    out = ph.fp8_matmul(one, sa[:1].expand(40, -1), b, sb, None, torch.float32)
    assert torch.equal(out, out[:1].expand(40, n)) and torch.allclose(out[0], want[0], rtol=1e-4, atol=float(want.abs().max()) * 1e-6)


def test_same_bits_again(dev):
    """No order of waves or workgroups changes a sum."""
    import torch

    for m, n, k, dtype in ((16, 4096, 4096, torch.bfloat16), (128, 4096, 16384, torch.bfloat16), (300, 1000, 12000, torch.float32),
                           (2000, 3000, 1024, torch.float16)):
        args = operands(m, m, n, k, dev)
        first = ph.fp8_matmul(*args, None, dtype)
        for _ in range(3):
            assert torch.equal(ph.fp8_matmul(*args, None, dtype).view(torch.uint8), first.view(torch.uint8))


def test_long_sums(dev):
    """K past every size of int8_matmul's: no limit but memory's."""
    import torch

    m, n, k = 20, 40, 200003
    args = operands(9, m, n, k, dev)
    check_large(ph.fp8_matmul(*args, None, torch.float32), *args, None, "float32")

"""What the products of 8-bit floats keep, in the units of their outputs: where 16-bit outputs are cut and by how much at
most, what that does to ordinary ones, and that 32-bit outputs count every product."""
import numpy as np
import pytest

import pyPhantom as ph
from test_gpu_clear_ops import dtype_of, f64, normal

pytestmark = pytest.mark.gpu

NARROW = ["bfloat16", "float16"]
# rows and columns that reach the streaming kernel and tiles
SIZES = [(1, 16), (5, 40), (130, 8300)]


def power(v):
    """A code's power of two as products are aligned by: that of its leading bit, 2^-6 for all below it."""
    return np.exp2(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6))))


def aligned_sum(a, b):
    """Products a b of one block as the 8-bit matrix instruction adds them: eight neighbours cut towards 0 at 2^-13 of the
    largest product of two powers (products that are 0 have none)."""
    total = 0.0
    for i in range(0, len(a), 8):
        x, y = a[i:i + 8], b[i:i + 8]
        at = np.where(x * y != 0, power(x) * power(y), 0.0).max()
        if at:
            total += np.trunc(x * y / at * 2.0 ** 13).sum() * at * 2.0 ** -13
    return total


def product(a, b, size, dtype, dev):
    """Every output of size[0] rows a and size[1] rows b, which are all the same number."""
    import torch

    m, n = size
    rows = [torch.tensor(v, dtype=torch.float32).to(torch.float8_e4m3fn).to(dev).expand(k, len(v)) for v, k in ((a, m), (b, n))]
    assert all(np.array_equal(f64(r[0].float()), v) for r, v in zip(rows, (a, b)))  # they are codes
    blocks = -(-len(a) // 128)
    one = torch.ones((), device=dev)
    out = ph.fp8_matmul(rows[0], one.expand(m, blocks), rows[1], one.expand(-(-n // 128), blocks), None, dtype_of(dtype))
    assert (out == out[0, 0]).all()
    return out[0, 0].item()


def crafted():
    """(name, a, b): blocks whose largest products cancel, so that what was cut beside them shows."""
    cases = []

    def put(name, pairs):
        a, b = np.zeros(128), np.zeros(128)
        for i, (x, y) in pairs.items():
            a[i], b[i] = x, y
        cases.append((name, a, b))

    for q in range(10):  # 2^q beside 2^16
        put(f"powers {q}", {0: (256, 256), 1: (2.0 ** (q - 4), 16), 8: (256, -256)})
        put(f"sevens {q}", {0: (256, 256), **{i: (-1.75 * 2.0 ** (q - 4), 15) for i in range(1, 8)}, 64: (-256, 256)})
        put(f"leading bits only {q}", {0: (480 - 32, 480 - 32), 1: (1.875 * 2.0 ** (q - 4), 16), 120: (448, -448)})
        put(f"far apart in the row {q}", {0: (256, 256), 8: (2.0 ** (q - 4), 16), 127: (256, -256)})
    for q in range(-3, 6):  # 2^q 2^-6 beside subnormal codes, which align like 2^-6
        put(f"subnormal a {q}", {0: (2.0 ** -9, 256), 3: (1.5 * 2.0 ** q, 2.0 ** -6), 16: (2.0 ** -9, -256)})
        put(f"subnormal b {q}", {9: (-256, 5 * 2.0 ** -9), 15: (2.0 ** -6, 1.125 * 2.0 ** q), 77: (256, 5 * 2.0 ** -9)})
        put(f"subnormal both {q}", {0: (2.0 ** -9, 2.0 ** -9), 1: (2.0 ** -9, 3 * 2.0 ** -9), 2: (2.0 ** q, 2.0 ** -6)})
        put(f"nothing beside it {q}", {0: (0, 448), 1: (448, 0), 2: (1.5 * 2.0 ** q, 2.0 ** -6)})
    return cases


@pytest.mark.parametrize("size", SIZES)
def test_cut(dev, size):
    """The rule that is stated, number by number; the sums of eights add up exactly in 32 bits here."""
    import torch

    for name, a, b in crafted():
        want = aligned_sum(a, b)
        for dtype in NARROW:
            rounded = torch.tensor(want, dtype=torch.float64).to(dtype_of(dtype)).item()
            assert product(a, b, size, dtype, dev) == rounded, (name, dtype, want)
        assert product(a, b, size, "float32", dev) == (a * b).sum(), name


@pytest.mark.parametrize("m,n,k", [(1, 512, 4096), (64, 512, 4096), (300, 700, 2050), (200, 2000, 1024)])
@pytest.mark.parametrize("dtype", NARROW)
def test_ordinary_outputs(dev, dtype, m, n, k):
    """States and weights as quantize_fp8 lays them out: the outputs' error against 64 bits is that of their rounding.
    Each of seven products loses less than 2^-13 P, P the largest of the eight products of powers: uniform and of
    products whose signs know nothing of each other (7 / 3)^(1/2) 2^-13 P in the mean square, beside a sum whose mean
    square is that of its products, P or more.  So a result is off by 1.53 2^-13 of itself.  A rounding to 8 bits is off by
    12^(-1/2) 2^-7 of a result's power of two, half of the result or more, to 11 bits by 12^(-1/2) 2^-10: together at most
    1.014 and 1.66 times the rounding's."""
    import torch

    a, sa = ph.quantize_fp8(normal(m + k, m, k, dtype="float32", dev=dev))
    b, sb = ph.quantize_fp8(normal(n + k, n, k, dtype="float32", dev=dev, spread=0.02), 128)
    got = ph.fp8_matmul(a, sa, b, sb, None, dtype_of(dtype)).double()
    wide = [c.float().double() * s.double().repeat_interleave(r, 0)[:c.shape[0]].repeat_interleave(128, 1)[:, :k]
            for c, s, r in ((a, sa, 1), (b, sb, 128))]
    want = torch.mm(wide[0], wide[1].t().contiguous())
    rounding = (want.to(dtype_of(dtype)).double() - want).norm()
    assert float((got - want).norm()) <= {"bfloat16": 1.014, "float16": 1.66}[dtype] * float(rounding)
    # and 32-bit outputs are the sums themselves: additions of 2^-24 of a sum, or of 2^-23 where the unit cuts
    full = ph.fp8_matmul(a, sa, b, sb, None, torch.float32).double()
    assert float((full - want).norm()) <= 2 * (k / 128 + 128) * 2.0 ** -24 * float(want.norm())

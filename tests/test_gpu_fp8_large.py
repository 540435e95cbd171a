"""Products of more outputs than low tiles cover in one launch: the first, the last and those at powers of two are where they
belong, everything else is 0."""
import pytest

import fp8_reference as R
import pfa_native as P
import pyPhantom as ph

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(1 << 28, 16), (1 << 26, 300), (1, 1 << 28), (5, (1 << 27) + 77)])
def test_most_outputs(dev, m, n):
    import torch

    k = 16
    rows, cols, _ = P.fp8_plan(m, n, k, 1)
    assert -(-m // (rows or 16)) * -(-n // cols) < 1 << 22
    a = torch.zeros((m, k), dtype=torch.uint8, device=dev)
    b = torch.zeros((n, k), dtype=torch.uint8, device=dev)
    # numbers of 1 to 8, in places of the rows that make products 1 and 0
    some_m = sorted({0, m - 1, m // 2, m // 3, min(m - 1, (1 << 25) + 3)})
    some_n = sorted({0, n - 1, n // 2, n // 3, min(n - 1, (1 << 26) + 5)})
    for i, r in enumerate(some_m):
        a[r, 0] = torch.tensor(1.0 + i).to(torch.float8_e4m3fn).view(torch.uint8)
    for i, c in enumerate(some_n):
        b[c, 0] = torch.tensor(1.0 + i).to(torch.float8_e4m3fn).view(torch.uint8)
    sa = torch.ones((m, 1), device=dev)
    sb = torch.ones((R.spans(n), 1), device=dev)
    sb[-1] = 0.5
    out = ph.fp8_matmul(a.view(torch.float8_e4m3fn), sa, b.view(torch.float8_e4m3fn), sb, None, torch.bfloat16)
    last = (n - 1) // 128
    for i, r in enumerate(some_m):
        for j, c in enumerate(some_n):
            assert out[r, c] == (1 + i) * (1 + j) * (0.5 if c // 128 == last else 1), (r, c)
    found = sum(int((part != 0).sum()) for part in out.view(-1).split(1 << 30))
    assert found == len(some_m) * len(some_n)

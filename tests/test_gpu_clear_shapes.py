"""Every kernel behind the clear operators against the definition in 64 bits, at sizes that the launch rules send to it
(clear_shapes.py; test_clear_shapes.py checks that they do)."""
import pytest

import clear_reference as R
import pfa_native as P
import pyPhantom as ph
from clear_shapes import PRODUCTS
from test_gpu_clear_ops import TYPES, U, codes_of, dtype_of, layouts, normal

pytestmark = pytest.mark.gpu


def lines(codes):
    """Rows at multiples of 128 bytes, as quantize_int8 lays its codes out."""
    import torch

    m, k = codes.shape
    return torch.full((m, -(-k // 128) * 128), 77, dtype=torch.int8, device=codes.device)[:, :k].copy_(codes)


def within(out, prod, bias, eps):
    """The sum is exact; its float, the two scales and the bias round once each, then the type does.  On the GPU, in 64
    bits."""
    want = prod if bias is None else prod + bias.double()
    slack = 4 * U * prod.abs() + (U + eps) * want.abs() * (1 + 2.0 ** -7) + 2.0 ** -24
    return bool(((out.double() - want).abs() <= slack).all())


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product_shapes(dev, m, n, k):
    import torch

    a, b = codes_of(m + k, m, k, dev, full=True), codes_of(n + k, n, k, dev, full=True)
    sa, sb = normal(1, m, dev=dev).abs() / 127, normal(2, n, dev=dev) / (127 * k ** 0.5)
    bias = normal(3, n, dev=dev)
    sums = torch.mm(a.double(), b.double().t().contiguous())  # whole numbers below 2^31: exact
    prod = sums * sa.double()[:, None] * sb.double()[None, :]
    for place in (layouts, "odd"), (layouts, "apart"), (lines,), (layouts, "dense"):
        x, y = place[0](a, *place[1:]), place[0](b, *place[1:])
        for name in TYPES:
            for add in (bias, None):
                out = ph.int8_matmul(x, sa, y, sb, add, dtype_of(name))
                assert within(out, prod, add, R.EPS[name]), (place, name, add is None)


@pytest.mark.parametrize("m,n,k", PRODUCTS[::5])
def test_product_stays_in_its_rows(dev, m, n, k):
    """Outputs in rows that are apart, at an odd address: nothing between them is written."""
    import torch

    a, b = codes_of(1, m, k, dev, "odd"), codes_of(2, n, k, dev, "odd")
    sa, sb = normal(1, m, dev=dev).abs() / 127, normal(2, n, dev=dev) / (127 * k ** 0.5)
    need = P.matmul_workspace(m, n, k)
    for code, name in enumerate(TYPES):
        want = ph.int8_matmul(a, sa, b, sb, None, dtype_of(name))
        big = torch.full((m, n + 3), -5.0, dtype=dtype_of(name), device=dev)
        space = torch.empty(need, dtype=torch.uint8, device=dev)
        P.call("pfa_int8_matmul", a.data_ptr(), a.stride(0), sa.data_ptr(), b.data_ptr(), b.stride(0), sb.data_ptr(),
               None, m, n, k, big[:, 1:].data_ptr(), code, n + 3, space.data_ptr() if need else None, need,
               P.stream_handle(torch.cuda.current_stream(dev)))
        assert torch.equal(big[:, 1:n + 1], want)
        assert (big[:, 0] == -5).all() and (big[:, n + 1:] == -5).all()

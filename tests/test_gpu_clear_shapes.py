"""Every kernel behind the clear operators against the definition in 64 bits, at sizes that the launch rules send to it
(clear_shapes.py; test_clear_shapes.py checks that they do)."""
import math

import numpy as np
import pytest

import clear_reference as R
import pfa_native as P
import pyPhantom as ph
from clear_shapes import PROBABILITIES, PRODUCTS, WIDE_ROWS
from test_gpu_clear_ops import TYPES, U, check_codes, check_probs, codes_of, dtype_of, f64, layouts, normal

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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", PROBABILITIES)
def test_probability_rows(dev, dtype, rows, vocab):
    """Rows in one piece, with everything that a row can hold in each call: masks, temperature 0 with a tie, NaN and
    infinities in masked and in allowed places, nothing allowed, the last vector of an odd row."""
    import torch

    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn((rows, vocab), generator=g) * 4).to(dtype_of(dtype))
    t = 0.3 + torch.rand(rows, generator=g)
    mask = torch.rand((rows, vocab), generator=g) < torch.rand((rows, 1), generator=g)
    last = vocab - 1
    x[0, 3], mask[0, 3], mask[0, last] = math.nan, False, True      # NaN in a masked place
    if rows > 10:
        t[1], x[1, last], x[1, 5], mask[1, last], mask[1, 5] = 0, 50., 50., True, True  # a tie at temperature 0
        mask[2] = False                                             # nothing allowed
        x[3] = -math.inf
        x[4, last], mask[4, last] = math.nan, True                  # NaN in an allowed place
        x[5, 7], mask[5, 7] = math.inf, True                        # infinity in an allowed place
        x[6, last], mask[6, last] = math.inf, False                 # infinity in a masked place
        t[7], x[7, 9], mask[7, 9] = 0, math.inf, True
        t[8] = math.nan
        mask[9], mask[9, last] = torch.tensor(False), True          # one place
    every = torch.ones(vocab, dtype=torch.bool)
    every[[3, 7, last - 1]] = False
    out, heat = torch.empty((rows, vocab), device=dev), t.to(dev)
    for k, m in enumerate((mask, every, None)):
        logits, there = layouts(x.to(dev), ("odd", "dense", "apart")[k]), None if m is None else m.to(dev)
        p = ph.token_probabilities(logits, heat, there)
        check_probs(p, f64(x), f64(t), None if m is None else m.numpy())
        # without a workspace the call is only possible in one piece
        P.call("pfa_token_probabilities", logits.data_ptr(), logits.stride(0) if rows > 1 else vocab, TYPES.index(dtype),
               rows, vocab, heat.data_ptr(), 1.0, None if m is None else there.data_ptr(),
               vocab if m is mask else 0, out.data_ptr(), None, 0, P.stream_handle(torch.cuda.current_stream(dev)))
        assert np.array_equal(f64(out), f64(p), equal_nan=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDE_ROWS)
def test_quantize_wide_rows(dev, dtype, width):
    import torch

    for rows in (1, 5):
        x = normal(width + rows, rows, width, dtype=dtype, dev=dev)
        for kind in ("dense", "apart", "odd"):
            codes, scales = ph.quantize_int8(layouts(x, kind))
            check_codes(codes, scales, f64(x), 0)
    x[1, width - 1], x[2, 0], x[3] = math.nan, math.inf, 0
    codes, scales = ph.quantize_int8(x)
    assert torch.isnan(scales[1:3]).all() and (codes[1:4] == 0).all() and scales[3] == 0
    check_codes(codes[[0, 4]], scales[[0, 4]], f64(x[[0, 4]]), 0)
    w, r = normal(1, width, dtype=dtype, dev=dev, spread=0.3), normal(2, 5, width, dtype=dtype, dev=dev)
    x = normal(3, 5, width, dtype=dtype, dev=dev)
    codes, scales, total = ph.rms_norm_int8(layouts(x, "odd"), w, 1e-5, r)
    check_codes(codes, scales, R.rms_norm(f64(x), f64(w), 1e-5, f64(r)), width / 64 + 20)
    assert torch.equal(total, (x.float() + r.float()).to(x.dtype))

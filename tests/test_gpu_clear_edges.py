"""Where the clear operators' 32 bits end, and the rules of their roundings, against the definitions."""
import math

import numpy as np
import pytest

import clear_reference as R
import pyPhantom as ph
from test_gpu_clear_ops import TYPES, check_codes, check_probs, dtype_of, f64, layouts, normal

pytestmark = pytest.mark.gpu

# reaches every kernel of the rows: a wave with and without whole vectors, 256 and 1024 threads, rows read twice
WIDTHS = [1, 5, 9, 300, 2047, 4096, 8190, 16384, 20003, 32770, 40001, 70000]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_of_tiny_rows(dev, dtype, width):
    """Squares that are subnormal or vanish in 32 bits, at an eps that does not hide them, beside ordinary rows."""
    import torch

    x, r = (normal(width + k, 7, width, dtype="float32", dev=dev, spread=0.1) for k in (0, 1))
    size = torch.tensor([1e-23, 1.0, 1e-30, 0.0, 1e-19, 1e-14, 1e-36], device=dev)[:, None]
    x, r = ((t * size).to(dtype_of(dtype)) for t in (x, r))
    w = normal(3, width, dtype=dtype, dev=dev, spread=0.1)
    for eps in (0.0, 1e-60, 1e-30):
        for res in (None, r):
            codes, scales, total = ph.rms_norm_int8(layouts(x, "odd"), w, eps, res)
            with np.errstate(all="ignore"):
                v = R.rms_norm(f64(x), f64(w), eps, None if res is None else f64(res))
            v[3] = 0  # a row of zeros
            check_codes(codes, scales, v, width / 64 + 20)
    # the smallest numbers there are
    whole = torch.randint(-900, 901, (3, width), generator=torch.Generator().manual_seed(width)).to(dev)
    whole[:, 0] = 900
    x = (whole.double() * 2.0 ** (-149 if dtype == "float32" else -133)).to(dtype_of(dtype))
    one = torch.ones(width, device=dev, dtype=x.dtype)
    codes, scales, _ = ph.rms_norm_int8(x, one, 0.0)
    check_codes(codes, scales, R.rms_norm(f64(x), f64(one), 0.0), width / 64 + 20)


def nearest(codes, v):
    """codes are 127 v / max|v| to the nearest, ties to even: exact in 64 bits (127 v and code max|v| have 31 bits)."""
    c, v = codes.double(), v.double()
    top = v.abs().amax(-1, keepdim=True)
    off = (127 * v - c * top).abs() * 2
    return bool(((off < top) | ((off == top) & (c % 2 == 0))).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_codes_are_the_nearest(dev, dtype, width):
    """Every code and every scale by the definition, bit for bit: many values, and many that stand on a tie (half the
    largest one is 63.5 steps)."""
    import torch

    rows = max(8, (1 << 21) // width)
    x = normal(width, rows, width, dtype=dtype, dev=dev, spread=0.2)
    top = x.abs().amax(-1)
    x[:, width // 2::5] = (top / 2)[:, None]
    x[::2, width // 3::7] = (-top / 2)[::2, None]
    x[:, 0] = top
    codes, scales = ph.quantize_int8(x)
    assert nearest(codes, x)
    # a quotient of 24 bits rounded from 53 is the one rounded at once
    assert torch.equal(scales, (x.double().abs().amax(-1) / 127).float())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_norm_has_the_quantizations_codes(dev, dtype, width):
    """The norm's factor is common to a row: its codes are those of (x + residual) weight, each rounded to 32 bits."""
    import torch

    rows = max(8, (1 << 21) // width)
    x, r = (normal(width + k, rows, width, dtype=dtype, dev=dev, spread=0.2) for k in (0, 1))
    w = normal(width, width, dtype=dtype, dev=dev, spread=0.2)
    codes, _, _ = ph.rms_norm_int8(x, w, 1e-6, r)
    y = (x.float() + r.float()) * w.float()
    assert torch.equal(codes, ph.quantize_int8(y)[0])
    assert nearest(codes, y)


@pytest.mark.parametrize("heat", [1e31, 1e38])
def test_large_temperatures(dev, heat):
    """A number means what a tensor of it means, up to the largest."""
    import torch

    x = normal(1, 4, 300, dev=dev) * 1e30
    p = ph.token_probabilities(x, heat)
    assert torch.equal(p, ph.token_probabilities(x, torch.full((4,), heat, device=dev)))
    check_probs(p, f64(x), np.full(4, float(np.float32(heat))), None)


@pytest.mark.parametrize("eps", [1e31, 1e39, 1e60])
def test_large_eps(dev, eps):
    """An eps past 32 bits leaves scales within them."""
    for width in (5, 300, 4096, 40001):
        x = normal(width, 3, width, dev=dev, spread=0.1) * 1e15
        w = normal(1, width, dev=dev, spread=0.1)
        codes, scales, _ = ph.rms_norm_int8(x, w, eps)
        assert (scales > 0).all()
        check_codes(codes, scales, R.rms_norm(f64(x), f64(w), eps), width / 64 + 20)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,vocab", [(4, 5), (4, 300), (4, 9000), (70, 20000), (4, 131072)])
def test_logits_of_the_types_range(dev, dtype, rows, vocab):
    """Differences of logits that pass 32 bits, at temperatures that bring them back, the infinite one among them."""
    import torch

    x = (normal(vocab, rows, vocab, spread=0) * 1e38).clamp_(-3.3e38, 3.3e38)
    x[:, 0], x[:, -1] = 3.3e38, -3.3e38
    x = x.to(dtype_of(dtype))
    mask = torch.rand((rows, vocab), generator=torch.Generator().manual_seed(1)) < 0.5
    mask[:, 0] = mask[:, -1] = True
    for heat in (1e37, 1e38, 2e38, math.inf):
        t = torch.full((rows,), heat)
        for m in (None, mask):
            p = ph.token_probabilities(x.to(dev), t.to(dev), None if m is None else m.to(dev))
            check_probs(p, f64(x), f64(t), None if m is None else m.numpy())


@pytest.mark.parametrize("rows,vocab", [(4, 5), (4, 300), (4, 9000), (70, 20000), (4, 131072)])
def test_subnormal_temperatures(dev, rows, vocab):
    """Temperatures and differences of logits below 2^-126, down to where log2(e) / t passes 32 bits."""
    import torch

    x = torch.randint(-20, 1, (rows, vocab), generator=torch.Generator().manual_seed(vocab)) * 1e-39
    x = x.to(torch.float32)
    for heat in (4.9e-39, 7e-39, 1e-38):
        t = torch.full((rows,), heat)
        # t and c have 22 bits or more here: a relative error of 2^-21 in exponents of up to 4.1
        p = f64(ph.token_probabilities(x.to(dev), t.to(dev)))
        want = R.probabilities(f64(x), f64(t))
        assert np.all(np.abs(p - want) <= (8.2 * 2.0 ** -21 + vocab / 64 * 2.0 ** -24) * want)

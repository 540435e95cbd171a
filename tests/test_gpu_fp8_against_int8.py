"""Which codes keep what: states with a few channels far larger than the others, through the norm and a product, in integer
codes with a scale a row and in 8-bit floats with a scale for each block of 128."""
import pytest

import pyPhantom as ph

pytestmark = pytest.mark.gpu

EPS = 1e-6
ROWS, WIDTH, OUT = 64, 4096, 512


def errors(dev, size, beside):
    """{codes: error of the product, relative, in the mean square}.  Every `beside`-th channel is `size` times the others and
    has no weight in the product; the weights are -1, 0 and 1, which both codes hold exactly."""
    import torch

    g = torch.Generator().manual_seed(int(size))
    x = torch.randn((ROWS, WIDTH), generator=g)
    x[:, ::beside] = size * torch.where(x[:, ::beside] < 0, -1.0, 1.0)
    b = torch.randint(-1, 2, (OUT, WIDTH), generator=g).float()
    b[:, ::beside] = 0
    b[:, 1] = 1  # no row of zeros
    x, b, gain = x.to(dev), b.to(dev), torch.ones(WIDTH, device=dev)
    y = x.double()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS)
    want = torch.mm(y, b.double().t().contiguous())
    found = {}
    for name, norm, product, weights in (("int8", ph.rms_norm_int8, ph.int8_matmul, ph.quantize_int8(b)),
                                         ("e4m3", ph.rms_norm_fp8, ph.fp8_matmul, ph.quantize_fp8(b, 128))):
        codes, scales, _ = norm(x, gain, EPS)
        got = product(codes, scales, *weights, None, torch.float32).double()
        found[name] = float((got - want).norm() / want.norm())
    return found


@pytest.mark.parametrize("beside", [128, 1024])
@pytest.mark.parametrize("size", [30, 100, 1000])
def test_channels_of_different_size(dev, size, beside):
    """Other channels have deviation 1, and a product of them with weights whose signs know nothing of theirs is off, in the
    mean square, by what its values are.  A floating code is off by 2^-4 of its value at most; below 2^-6 scales (scale
    < 2 size / 448) by 2^-10 scales, less than size 2^-18.  An integer code is a multiple of size / 127: where
    that is 30 / 127 the step's 12^-1/2 part is more than 2^-4 (.068), and from 100 on rounding to it is off by more than
    .22; of values below size / 254, 3.9 deviations at 1000, nothing is left."""
    found = errors(dev, size, beside)
    assert found["e4m3"] <= 2.0 ** -4 + size * 2.0 ** -18
    assert found["int8"] > {30: 2.0 ** -4, 100: 0.2, 1000: 0.95}[size]


def test_channels_of_one_size(dev):
    """Here integer codes are the closer ones: a step of max / 127, max below 6 deviations, against 4 bits of each value."""
    found = errors(dev, 1, 128)
    assert found["int8"] <= 6 / 127 / 12 ** 0.5 * 1.05 < 0.02
    assert 0.02 < found["e4m3"] <= 2.0 ** -4

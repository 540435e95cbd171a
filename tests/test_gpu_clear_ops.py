"""The clear end of an encrypted generation step on the GPU, against numpy in 64 bits
(clear_reference.py).  Tolerances follow from the operations' roundings; they stand beside
each comparison."""
import math

import numpy as np
import pytest

import clear_reference as R
import pyPhantom as ph

pytestmark = pytest.mark.gpu

TYPES = ["float32", "bfloat16", "float16"]
U = 2.0 ** -24  # one rounding to 32 bits, relative


def dtype_of(name):
    import torch

    return getattr(torch, name)


def normal(seed, *shape, dtype="float32", dev=None, spread=1.0):
    """Normal values in `dtype`, rows and columns of different size."""
    import torch

    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[-1], generator=g))
    if len(shape) > 1:
        x = x * torch.exp(spread * torch.randn((*shape[:-1], 1), generator=g))
    return x.to(dtype_of(dtype)).to(dev)


def f64(t):
    return t.detach().cpu().double().numpy()


def layouts(t, kind):
    """The same values in other memory: rows apart, rows off every alignment."""
    import torch

    if kind == "dense":
        return t
    pad = 5 if kind == "odd" else 16
    off = 1 if kind == "odd" else 8
    big = torch.zeros((*t.shape[:-1], t.shape[-1] + pad), dtype=t.dtype, device=t.device)
    view = big[..., off:off + t.shape[-1]]
    view.copy_(t)
    return view


# ------------------------------------------------------------- codes
WIDTHS = [1, 2, 7, 16, 63, 64, 65, 100, 255, 257, 1000, 1024, 2050, 4096, 5119, 8192, 16384, 20003, 70000]


def check_codes(codes, scales, v, sum_terms):
    """v in 64 bits.  A code is rint of 127 v / max: the value has at most 8 roundings (residual, gain, factor,
    product, the row's lift), so it is within 127 * 8 U of the exact one, and a code within half a step more.  A scale
    has 4, and half of those of a sum of squares of `sum_terms` terms one after the other."""
    real, want = R.quantized(v)
    c, s = f64(codes), f64(scales)
    assert c.shape == v.shape and s.shape == v.shape[:-1]
    assert np.all(np.abs(c - real) <= 0.5 + 127 * 8 * U)
    assert np.all(np.abs(s - want) <= (8 + sum_terms / 2) * U * want + 2.0 ** -148)
    assert np.all(np.abs(c) <= 127)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_quantize(dev, dtype, width):
    for rows in (1, 3, 37):
        x = normal(width + rows, rows, width, dtype=dtype, dev=dev)
        for kind in ("dense", "apart", "odd"):
            codes, scales = ph.quantize_int8(layouts(x, kind))
            check_codes(codes, scales, f64(x), 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("width", WIDTHS)
def test_norm(dev, dtype, width):
    import torch

    for rows in (1, 3, 37):
        x, r = (normal(width + rows + k, rows, width, dtype=dtype, dev=dev) for k in (0, 50000))
        w = normal(width, width, dtype=dtype, dev=dev, spread=0.3)
        for kind in ("dense", "apart", "odd"):
            for res in (None, r):
                args = layouts(x, kind), layouts(w, kind), 1e-5, None if res is None else layouts(res, kind)
                codes, scales, total = ph.rms_norm_int8(*args)
                v = R.rms_norm(f64(x), f64(w), 1e-5, None if res is None else f64(res))
                # a thread of 64 or more on a row, then a tree
                check_codes(codes, scales, v, width / 64 + 20)
                if res is None:
                    assert total is args[0]
                else:  # one rounding to 32 bits, one to the type: what torch does
                    assert torch.equal(total, (x.float() + r.float()).to(x.dtype))


def test_quantize_edges(dev):
    """Rows of zeros, one element, subnormals, the largest numbers, NaN and infinities in one call."""
    import torch

    inf, nan = math.inf, math.nan
    rows = [[0.0] * 9, [0, 0, -3, 0, 0, 0, 0, 0, 0], [1e-45, -1e-45, 0, 0, 0, 0, 0, 0, 3e-45],
            [1e-38, -5e-39, 2e-39, 0, 0, 0, 0, 0, 0], [3.4e38, -3.4e38, 1e38, 1e37, 0, 0, 0, 0, 1],
            [nan, 1, 2, 3, 4, 5, 6, 7, 8], [1, 2, 3, 4, inf, 5, 6, 7, 8], [1, 2, 3, 4, 5, 6, 7, 8, -inf],
            [127, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -126.5], [1, 2, 3, inf, 5, nan, 7, 8, 9]]
    x = torch.tensor(rows, device=dev)
    codes, scales = ph.quantize_int8(x)
    bad = [5, 6, 7, 9]
    fine = [i for i in range(len(rows)) if i not in bad]
    check_codes(codes[fine], scales[fine], f64(x[fine]), 0)
    assert torch.isnan(scales[bad]).all() and (codes[bad] == 0).all()
    assert scales[0] == 0 and (codes[0] == 0).all()
    # halves of a step go to the even code
    assert codes[8].tolist() == [127, 0, 2, 2, 0, -2, -2, 126, -126]


def test_norm_edges(dev):
    import torch

    inf, nan = math.inf, math.nan
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.ones((8, 300), device=dev, dtype=dtype)
        r = torch.ones_like(x)
        w = torch.ones(300, device=dev, dtype=dtype)
        x[0], r[0] = 0, 0       # a row of zeros: eps keeps the norm finite
        x[1], r[1] = 5, -5      # the residual takes everything away
        x[2, 17] = nan
        x[3, 299] = inf
        r[4, 0], x[4, 0] = -inf, inf
        x[5], r[5] = 1e30, 0    # squares pass 32 bits
        codes, scales, total = ph.rms_norm_int8(x, w, 1e-6, r)
        assert (codes[:2] == 0).all() and (scales[:2] == 0).all() and (total[:2] == 0).all()
        assert torch.isnan(scales[2:6]).all() and (codes[2:6] == 0).all()
        assert (codes[6:] == 127).all()
        # (2 / sqrt(4 + eps)) / 127
        assert (scales[6:] - 1 / 127).abs().max() < 1e-8
        codes, scales, _ = ph.rms_norm_int8(x[:1] * 0, w, 0.0)  # nothing at all, not even eps
        assert (codes == 0).all() and (scales == 0).all()
        w[3] = nan  # a gain that is no number reaches every row
        codes, scales, total = ph.rms_norm_int8(x, w, 1e-6, r)
        assert torch.isnan(scales).all() and (codes == 0).all()
        assert not torch.isnan(total[6:]).any()


def test_codes_shapes(dev):
    """Leading dimensions, no rows, empty rows, one row over and over, codes' alignment."""
    import torch

    x = normal(1, 2, 3, 4, 50, dev=dev)
    codes, scales = ph.quantize_int8(x)
    assert codes.shape == x.shape and scales.shape == (2, 3, 4)
    assert all(s % 16 == 0 for s in codes.stride()[:-1]) and codes.data_ptr() % 16 == 0
    check_codes(codes.reshape(24, 50), scales.reshape(24), f64(x).reshape(24, 50), 0)
    codes, scales = ph.quantize_int8(x[0, 0, 0])
    assert codes.shape == (50,) and scales.shape == ()
    check_codes(codes, scales, f64(x[0, 0, 0]), 0)
    turned = x.permute(1, 0, 2, 3)
    codes, scales = ph.quantize_int8(turned)
    check_codes(codes.reshape(24, 50), scales.reshape(24), f64(turned).reshape(24, 50), 0)
    codes, scales = ph.quantize_int8(x[:, :0])
    assert codes.shape == (2, 0, 4, 50) and scales.shape == (2, 0, 4)
    codes, scales = ph.quantize_int8(x[..., :0])
    assert codes.shape == (2, 3, 4, 0) and (scales == 0).all()
    w = normal(2, 50, dev=dev)
    codes, scales, total = ph.rms_norm_int8(x, w, 1e-6, x)
    assert total.shape == x.shape and scales.shape == (2, 3, 4)
    codes, scales, total = ph.rms_norm_int8(x[:0], w, 1e-6, x[:0])
    assert codes.shape == (0, 3, 4, 50) and total.shape == codes.shape
    same = x[0, 0, 0].expand(7, 50)
    codes, scales = ph.quantize_int8(same)
    check_codes(codes, scales, f64(same), 0)


# ------------------------------------------------------------- product
def codes_of(seed, rows, k, dev, layout="dense", full=False):
    import torch

    g = torch.Generator().manual_seed(seed)
    lo = -128 if full else -127
    return layouts(torch.randint(lo, 128, (rows, k), generator=g, dtype=torch.int8).to(dev), layout)


def check_product(out, a, sa, b, sb, bias):
    """The sum is exact; its float, the two scales and the bias round once each, then the type does."""
    name = str(out.dtype).split(".")[1]
    prod = (f64(a) @ f64(b).T) * f64(sa)[:, None] * f64(sb)[None, :]
    want = prod + (0 if bias is None else f64(bias))
    got = f64(out)
    assert got.shape == want.shape
    slack = 4 * U * np.abs(prod) + (U + R.EPS[name]) * np.abs(want) * (1 + 2.0 ** -7) + 2.0 ** -24
    assert np.all(np.abs(got - want) <= slack)


SHAPES = [(1, 1, 1), (1, 5, 16), (2, 3, 17), (1, 64, 64), (1, 1000, 4096), (3, 129, 2050), (5, 257, 128), (8, 4096, 512),
          (15, 300, 1000), (16, 512, 4095), (17, 100, 130), (20, 5000, 256), (31, 64, 8192), (33, 65, 63),
          (48, 1024, 640), (63, 777, 1023), (64, 64, 64), (65, 127, 129), (100, 200, 300), (127, 255, 384),
          (128, 128, 128), (129, 383, 515), (200, 1000, 96), (256, 256, 256), (257, 511, 2050), (300, 640, 1024),
          (512, 512, 512), (513, 1025, 127), (777, 503, 250), (1024, 768, 256), (1030, 1300, 640)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(dev, m, n, k):
    for i, layout in enumerate(("dense", "apart", "odd")):
        a, b = codes_of(m + n, m, k, dev, layout), codes_of(m + n + 1, n, k, dev, layout)
        sa = normal(1, m, dev=dev).abs() / 127
        sb = normal(2, n, dev=dev) / (127 * k ** 0.5)
        bias = normal(3, n, dev=dev) if i != 1 else None
        for dtype in TYPES:
            check_product(ph.int8_matmul(a, sa, b, sb, bias, dtype_of(dtype)), a, sa, b, sb, bias)


@pytest.mark.parametrize("m", [1, 2, 16, 20, 64, 130, 300])
def test_product_extremes(dev, m):
    """The largest sums that 32 bits hold: K = 131071 products of -128 and -128, and of -128 and 127."""
    import torch

    k, n = 131071, 70
    a = torch.full((m, k), -128, dtype=torch.int8, device=dev)
    b = torch.full((n, k), -128, dtype=torch.int8, device=dev)
    b[::2] = 127
    one = torch.ones(max(m, n), device=dev)
    out = ph.int8_matmul(a, one[:m], b, one[:n], None, torch.float32)
    assert (out[:, 1::2] == float(128 * 128 * k)).all()
    assert (out[:, ::2] == float(-128 * 127 * k)).all()


def test_product_edges(dev):
    """Nothing to sum, nothing to form, scales that are no numbers, leading dimensions, one row over and over."""
    import torch

    a, b = codes_of(1, 6, 40, dev), codes_of(2, 9, 40, dev)
    sa, sb, bias = normal(3, 6, dev=dev), normal(4, 9, dev=dev), normal(5, 9, dev=dev)
    assert torch.equal(ph.int8_matmul(a[:, :0], sa, b[:, :0], sb, bias, torch.float32), bias.expand(6, 9))
    assert (ph.int8_matmul(a[:, :0], sa, b[:, :0], sb) == 0).all()
    assert ph.int8_matmul(a[:0], sa[:0], b, sb).shape == (0, 9)
    assert ph.int8_matmul(a, sa, b[:0], sb[:0]).shape == (6, 0)
    sa[2], sb[3] = math.nan, math.inf
    out = ph.int8_matmul(a, sa, b, sb, None, torch.float32)
    assert torch.isnan(out[2]).all()
    keep = [0, 1, 3, 4, 5]
    other = [0, 1, 2, 4, 5, 6, 7, 8]
    assert not torch.isfinite(out[keep][:, 3]).any()
    check_product(out[keep][:, other].contiguous(), a[keep], sa[keep], b[other], sb[other], None)
    sa, sb = normal(3, 6, dev=dev), normal(4, 9, dev=dev)
    lead = ph.int8_matmul(a.view(2, 3, 40), sa.view(2, 3), b, sb, bias, torch.float32)
    flat = ph.int8_matmul(a, sa, b, sb, bias, torch.float32)
    assert lead.shape == (2, 3, 9) and torch.equal(lead.view(6, 9), flat)
    assert torch.equal(ph.int8_matmul(a[4], sa[4], b, sb, bias, torch.float32), flat[4])
    same = a[0].expand(6, 40)
    assert torch.equal(ph.int8_matmul(same, sa, b, sb, bias, torch.float32),
                       ph.int8_matmul(same.contiguous(), sa, b, sb, bias, torch.float32))


@pytest.mark.parametrize("m", [1, 40, 200])
def test_product_long(dev, m):
    """Offsets past 32 bits: 4.6 GB of weights; columns from both ends and the middle are checked."""
    import torch

    k, n = 32768, 140001
    b = torch.empty((n, k), dtype=torch.int8, device=dev)
    pick = [0, 1, 65535, 65536, 131071, 131072, 139999, 140000]
    b.zero_()
    b[pick] = codes_of(1, len(pick), k, dev)
    a = codes_of(2, m, k, dev)
    sa, sb = normal(3, m, dev=dev), normal(4, n, dev=dev)
    out = ph.int8_matmul(a, sa, b, sb, None, torch.float32)
    check_product(out[:, pick].contiguous(), a, sa, b[pick], sb[pick], None)
    assert int((out != 0).any(0).sum()) == len(pick)


def test_product_is_the_layers(dev):
    """A layer from its floating weights: quantized channels and tokens give the layer's output to 8 bits."""
    import torch

    x, w = normal(1, 33, 512, dev=dev, spread=0), normal(2, 200, 512, dev=dev, spread=0)
    (a, sa), (b, sb) = ph.quantize_int8(x), ph.quantize_int8(w)
    out = f64(ph.int8_matmul(a, sa, b, sb, None, torch.float32))
    want = f64(x) @ f64(w).T
    # each code is off by up to half a step of its row: sum over k of |x| sb / 2 + |w| sa / 2 + sa sb / 4
    slack = (np.abs(f64(x)).sum(1)[:, None] * f64(sb) + f64(sa)[:, None] * np.abs(f64(w)).sum(1)) / 2 + \
        512 * f64(sa)[:, None] * f64(sb) / 4
    assert np.all(np.abs(out - want) <= slack * 1.001)


# ------------------------------------------------------------- probabilities
VOCABS = [1, 2, 3, 31, 64, 65, 1000, 1023, 4096, 5003, 8192, 20000, 32768, 50001, 100003, 131072, 200001]


def check_probs(p, logits, temperature, mask, z=None):
    """p = exp((l - m) / T) / sum.  The exponent t has at most 4 roundings, so e^t is off by |t| 4 U and by 2 U of its
    own; the sum by as much at its terms' mean and V / 64 + 20 roundings; the quotient by 3."""
    got, want = f64(p), R.probabilities(logits, temperature, mask)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    for g, w, t in zip(got, want, temperature):
        if np.isnan(w).any() or t == 0:
            assert np.array_equal(g, w, equal_nan=True)
            continue
        with np.errstate(all="ignore"):
            size = np.where(w > 0, np.abs(np.log(w / max(w.max(), 1e-300))), 0)
        mean = (size * w).sum()
        slack = (4 * size + 4 * mean + len(w) / 64 + 40) * U * w + 2.0 ** -125
        assert np.all(np.abs(g - w) <= slack)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_probabilities(dev, dtype, vocab):
    import torch

    g = torch.Generator().manual_seed(vocab)
    for rows in (1, 3, 40):
        x = (torch.randn((rows, vocab), generator=g) * 4).to(dtype_of(dtype))
        t = (0.3 + torch.rand(rows, generator=g))
        t[0] = 1
        if rows > 1:
            t[1] = 0
        every = torch.rand((rows, vocab), generator=g) < torch.rand((rows, 1), generator=g)
        for k, mask in enumerate((None, every, every[rows // 2])):
            logits = layouts(x.to(dev), ("dense", "apart", "odd")[k])
            m = None if mask is None else layouts(mask.to(dev), "odd" if k == 2 else "dense")
            p = ph.token_probabilities(logits, t.to(dev), m)
            assert p.dtype == torch.float32
            check_probs(p, f64(x), f64(t), None if mask is None else mask.numpy())
        p = ph.token_probabilities(x.to(dev), 0.7)
        check_probs(p, f64(x), np.full(rows, 0.7), None)


@pytest.mark.parametrize("vocab", [9, 1000, 40000, 131072])
def test_probabilities_edges(dev, vocab):
    """Masks that leave nothing, masks by the type's lowest value, infinities and NaN in masked and allowed places,
    ties, temperatures at the ends."""
    import torch

    inf, nan = math.inf, math.nan
    x = torch.randn((16, vocab), generator=torch.Generator().manual_seed(1))
    t = torch.ones(16)
    mask = torch.ones((16, vocab), dtype=torch.bool)
    last = vocab - 1
    mask[0] = False                                     # nothing allowed
    mask[1], mask[1, last] = torch.tensor(False), True  # one place
    x[2] = -inf                                         # nothing by the logits
    x[3], x[3, 5] = torch.tensor(-inf), 2.0             # one place by the logits
    x[4], x[4, 1] = torch.finfo(torch.float32).min, 0.  # masked by the lowest number
    x[5] = torch.finfo(torch.float32).min               # everything so
    x[6, 3], mask[6, 3] = nan, False                    # NaN in a masked place
    x[7, last], mask[7, last] = inf, False              # infinity in a masked place
    x[8, last] = nan                                    # NaN in an allowed place
    x[9, 2] = inf                                       # infinity in an allowed place
    x[10, 4], x[10, last], t[10] = 50., 50., 0          # a tie at temperature 0
    x[11, 4], t[11] = inf, 0                            # infinity at temperature 0
    x[12, 6], t[12] = nan, 0                            # NaN at temperature 0
    t[13] = -1                                          # no temperature
    t[14] = nan
    t[15] = 1e-30                                       # one place takes all
    mask[11, 0] = mask[13, 0] = mask[14, 0] = False
    p = ph.token_probabilities(x.to(dev), t.to(dev), mask.to(dev))
    check_probs(p[:15], f64(x)[:15], f64(t)[:15], mask.numpy()[:15])
    assert p[15].sum() == 1 and int(p[15].argmax()) == int(x[15].argmax())
    assert p[10, 4] == 1 and p[11, 4] == 1
    # no probability outside, nothing from one row in another
    assert (p[~mask.to(dev)] == 0).all()
    # float32's lowest number is -infinity in bfloat16, bfloat16's own is not
    q = ph.token_probabilities(x[4:6].to(dev).to(torch.bfloat16), 0)
    assert q[0, 1] == 1 and q.sum() == 1
    low = torch.full((2, vocab), torch.finfo(torch.bfloat16).min, dtype=torch.bfloat16, device=dev)
    low[1, last] = 0
    for t in (0, 1.0):
        check_probs(ph.token_probabilities(low, t), f64(low), np.full(2, float(t)), None)


def test_probabilities_shapes(dev):
    import torch

    x = normal(1, 2, 3, 100, dev=dev)
    t = torch.rand((2, 3), device=dev) + 0.5
    mask = torch.rand((2, 3, 100), device=dev) < 0.5
    p = ph.token_probabilities(x, t, mask)
    assert p.shape == (2, 3, 100)
    check_probs(p.view(6, 100), f64(x).reshape(6, 100), f64(t).reshape(6), mask.cpu().numpy().reshape(6, 100))
    p = ph.token_probabilities(x[1, 2])
    check_probs(p.view(1, 100), f64(x[1, 2])[None], np.ones(1), None)
    assert ph.token_probabilities(x[:0]).shape == (0, 3, 100)
    assert ph.token_probabilities(x[..., :0]).shape == (2, 3, 0)
    row = x[0, 0].expand(5, 100)
    check_probs(ph.token_probabilities(row, 2.0), f64(row), np.full(5, 2.0), None)
    allow = mask[0, 0].expand(5, 100)
    check_probs(ph.token_probabilities(row, 2.0, allow), f64(row), np.full(5, 2.0), allow.cpu().numpy())


# ------------------------------------------------------------- drafts
def drafts_case(seed, batch, drafts, vocab, dtype="float32", near=0.5):
    import torch

    g = torch.Generator().manual_seed(seed)
    logits = 2 * torch.randn((batch, drafts + 1, vocab), generator=g)
    p = torch.softmax(logits, -1).to(dtype_of(dtype))
    q = torch.softmax(logits[:, :drafts] + near * torch.randn((batch, drafts, vocab), generator=g), -1)
    x = (q / -torch.log1p(-torch.rand(q.shape, generator=g))).argmax(-1) if drafts else \
        torch.zeros((batch, 0), dtype=torch.int64)
    u = torch.rand((batch, drafts), generator=g)
    e = -torch.log1p(-torch.rand((batch, vocab), generator=g)) + 1e-10
    n = torch.randint(0, drafts + 1, (batch,), generator=g)
    return x, p, u, e, q.to(p.dtype), n


def check_drafts(dev, x, p, u, e, q=None, n=None):
    import torch

    got = ph.verify_drafts(*(None if t is None else t.to(dev) for t in (x, p, u, e, q, n)))
    want = R.verify(x.numpy(), f64(p), f64(u), f64(e), None if q is None else f64(q),
                    None if n is None else n.numpy())
    assert got[0].dtype == x.dtype and got[1].dtype == torch.int32
    assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1])
    return got


@pytest.mark.parametrize("batch,drafts,vocab", [
    (1, 0, 1), (1, 1, 1), (1, 4, 7), (3, 2, 64), (5, 3, 1000), (1, 4, 32768), (2, 8, 50001), (64, 5, 1023), (300, 2, 130),
    (1, 0, 131072), (1, 3, 131072), (9, 1, 100003), (40, 3, 20000), (2, 70, 50), (1, 300, 9)])
def test_verify(dev, batch, drafts, vocab):
    import torch

    for dtype in TYPES:
        x, p, u, e, q, n = drafts_case(batch + drafts + vocab, batch, drafts, vocab, dtype)
        check_drafts(dev, x, p, u, e, q)
        check_drafts(dev, x.to(torch.int32), p, u, e, q, n)
        check_drafts(dev, x, p, u, e, None, n.to(torch.int32))
        # every draft kept, and none
        check_drafts(dev, x, p, torch.zeros_like(u), e, q)
        check_drafts(dev, x, p, torch.full_like(u, 2.0), e, q)


def test_verify_layouts(dev):
    """Probabilities and noise out of larger tensors; lengths outside their range are clamped."""
    import torch

    x, p, u, e, q, n = drafts_case(3, 6, 4, 501)
    want = check_drafts(dev, x, p, u, e, q)
    dp, dq = p.to(dev), q.to(dev)
    big = torch.zeros((6, 9, 520), device=dev)
    big[:, 1:6, 3:504] = dp
    more = torch.zeros((4, 6, 501), device=dev)
    more.copy_(dq.transpose(0, 1))
    got = ph.verify_drafts(x.to(dev), big[:, 1:6, 3:504], u.to(dev), layouts(e.to(dev), "odd"), more.transpose(0, 1))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    check_drafts(dev, x, p, u, e, q, torch.tensor([-3, 99, 0, 4, 2, 1 << 40]))
    shared = e[:1].expand(6, 501)
    check_drafts(dev, x, p, u, shared, q)


@pytest.mark.parametrize("vocab", [5, 40000])
def test_verify_edges(dev, vocab):
    """Tokens outside the vocabulary, equal distributions, empty targets, one-hot targets, zero noise, NaN."""
    import torch

    x, p, u, e, q, n = drafts_case(11, 12, 3, vocab)
    x[0, 1], x[1, 0], x[2, 2] = -1, vocab, 1 << 40
    q[3], u[3] = p[3, :3], 1.5                 # equal, yet refused: nothing left over, the target itself
    p[4] = 0                                   # a target that allows nothing
    p[5] = 0
    p[5, torch.arange(4), x[5, [0, 1, 2, 0]]] = 1.0   # a greedy target that agrees
    p[6] = 0
    p[6, :, vocab - 1] = 1.0                   # a greedy target that does not
    x[6], u[6] = 0, 0.5
    q[7, 0, x[7, 0]] = 0.0                     # a draft its own model ruled out
    e[8, 3] = 0.0                              # no noise: the weight wins
    p[9, 0, x[9, 0]] = math.nan                # not kept, not drawn
    p[9, 0, 2] = math.nan
    u[10, 0] = math.nan
    q[11, 0] = math.nan
    check_drafts(dev, x, p, u, e, q)
    check_drafts(dev, x, p, u, e, None)
    # equal weights: the lowest
    flat = torch.full((1, 1, vocab), 1 / vocab)
    none = torch.zeros((1, 0), dtype=torch.int64)
    got = ph.verify_drafts(none.to(dev), flat.to(dev), torch.zeros((1, 0), device=dev), torch.ones((1, vocab), device=dev))
    assert got[0].tolist() == [[0]] and got[1].tolist() == [0]
    got = ph.verify_drafts(none.to(dev)[:0], flat.to(dev)[:0], torch.zeros((0, 0), device=dev),
                           torch.ones((0, vocab), device=dev))
    assert got[0].shape == (0, 1) and got[1].shape == (0,)


def test_verify_distribution(dev):
    """The first token, kept or drawn, is distributed as the target says, and so is the second after each first."""
    import torch

    batch, vocab = 400000, 6
    g = torch.Generator(device=dev).manual_seed(5)
    p0 = torch.tensor([0.05, 0.3, 0.1, 0.25, 0.2, 0.1], device=dev)
    q0 = torch.tensor([0.3, 0.1, 0.1, 0.1, 0.1, 0.3], device=dev)
    p1 = torch.tensor([0.5, 0.1, 0.1, 0.1, 0.1, 0.1], device=dev)
    draw = lambda w, *shape: (w / torch.empty((*shape, vocab), device=dev).exponential_(generator=g)).argmax(-1)  # noqa: E731
    x = draw(q0, batch, 1)
    p = torch.stack([p0, p1]).expand(batch, 2, vocab)
    q = q0.expand(batch, 1, vocab)
    u = torch.rand((batch, 1), device=dev, generator=g)
    e = torch.empty((batch, vocab), device=dev).exponential_(generator=g)
    tokens, accepted = ph.verify_drafts(x, p, u, e, q)
    for place, want in ((0, p0), (1, p1)):
        seen = tokens[:, place]
        seen = seen[seen >= 0]
        share = torch.bincount(seen, minlength=vocab).double() / seen.numel()
        # five standard deviations of each share
        assert ((share - want.double()).abs() < 5 * (want.double() * (1 - want.double()) / seen.numel()).sqrt()).all()
    keep = float(accepted.double().mean())
    overlap = float(torch.minimum(p0, q0).sum())
    assert abs(keep - overlap) < 5 * math.sqrt(overlap * (1 - overlap) / batch)


# ------------------------------------------------------------- streams, graphs, together
def step(x, r, w, b, sb, drafts, u, e):
    """Hidden states of batch x places to tokens, as the holder of the key runs it."""
    codes, scales, total = ph.rms_norm_int8(x, w, 1e-6, r)
    import torch

    logits = ph.int8_matmul(codes, scales, b, sb, None, torch.float32)
    p = ph.token_probabilities(logits, 0.8)
    return (*ph.verify_drafts(drafts, p, u, e), p, total)


def step_inputs(dev, seed, batch=3, drafts=4, width=512, vocab=20000):
    import torch

    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn((batch, drafts + 1, width), device=dev, generator=g).to(torch.bfloat16)
    r = torch.randn((batch, drafts + 1, width), device=dev, generator=g).to(torch.bfloat16)
    w = torch.ones(width, device=dev, dtype=torch.bfloat16)
    b, sb = ph.quantize_int8(torch.randn((vocab, width), device=dev, generator=g) * 0.1)
    d = torch.randint(0, vocab, (batch, drafts), device=dev, generator=g)
    u = torch.rand((batch, drafts), device=dev, generator=g)
    e = torch.empty((batch, vocab), device=dev).exponential_(generator=g)
    return x, r, w, b, sb, d, u, e


def test_step_on_other_streams(dev):
    """The same step on two side streams at once gives what the default stream gives."""
    import torch

    ins = [step_inputs(dev, s) for s in (1, 2)]
    want = [step(*i) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = [None, None]
    for _ in range(5):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = step(*ins[k])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_step_in_a_graph(dev):
    """The step captured, replayed several times on changing inputs with eager work between the replays."""
    import torch

    ins = step_inputs(dev, 3)
    step(*ins)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*ins)
    for seed in (4, 5, 6, 7):
        fresh = step_inputs(dev, seed)
        for a, b in zip(ins, fresh):
            a.copy_(b)
        want = step(*ins)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        eager = step(*fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager))


def test_same_call_same_bits(dev):
    """No sum depends on the order in which workgroups end."""
    import torch

    for ins in (step_inputs(dev, 8), step_inputs(dev, 9, batch=1, vocab=131072), step_inputs(dev, 9, batch=60)):
        want = step(*ins)
        for _ in range(5):
            assert all(torch.equal(a, b) for a, b in zip(step(*ins), want))


def test_example(dev):
    """examples/encrypted_decoding.py: an encrypted layer between drafts and their check."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "encrypted_decoding.py")
    spec = importlib.util.spec_from_file_location("encrypted_decoding", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    text, worst = module.run(rounds=2, say=lambda _: None)
    assert 2 <= len(text) <= 10 and all(0 <= t < 1000 for t in text)
    # codes are off by half a step of 1/127 of their row's largest, about 4 deviations: logits of deviation 1 by
    # 0.013 (normal) in each factor, so probabilities by 0.02 / 0.8, half of it in total variation
    assert worst < 0.03

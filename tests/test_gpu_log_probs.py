"""Log probabilities of given tokens, entropy and alternatives on the GPU, against numpy in 64 bits (fp8_reference.py).
Alternatives are compared place by place; tolerances follow from the operations' roundings."""
import math

import numpy as np
import pytest

import fp8_reference as R
import pyPhantom as ph
from test_gpu_clear_ops import TYPES, dtype_of, f64, layouts

pytestmark = pytest.mark.gpu

U = R.U


def logits_of(seed, rows, vocab, dtype, dev, spread=3.0):
    import torch

    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g) * spread).to(dtype_of(dtype)).to(dev)


def check(got, logits, tokens, top, temperature=1.0, mask=None):
    """An exponent g has 3 roundings and its base's (4 U |g|), a weight 2 more, and a thread adds its weights one after the
    other (vocab / 256 of them, 3 roundings more for each vector that lifts its base), then 12 in a tree and as many
    stretches as there are: `terms`.  So log S is off by U (4 H + 5 + terms) (H >= sum p |d|), and one rounding of
    its own; d has 3.  The mean of g has the weights' errors once more, in sum p |d| and sum p d^2."""
    rows = logits.reshape(-1, logits.shape[-1])
    n, vocab = rows.shape
    t = np.broadcast_to(f64(temperature) if hasattr(temperature, "cpu") else np.float32(temperature), (n,)).reshape(-1)
    m = None if mask is None else mask.cpu().numpy().reshape(-1, vocab) if mask.dim() > 1 else mask.cpu().numpy()
    x = tokens.cpu().numpy().reshape(n, -1)
    given, entropy, tops, places, moments = R.log_probs(f64(rows), x, top, t, m)
    # what passes 32 bits is -infinity there
    given, tops = (np.where(v < -3.4028235677973366e38, -np.inf, v) for v in (given, tops))
    assert got[0].shape == tokens.shape and got[1].shape == logits.shape[:-1] and got[2].shape == (*logits.shape[:-1], top)
    assert got[3].dtype == tokens.dtype and np.array_equal(got[3].cpu().numpy().reshape(n, top), places)
    terms = vocab / 256 * 1.4 + 40
    d1, d2, log_s = moments.T
    room = U * (4 * d1 + 6 + terms + 2 * log_s)
    for a, want in ((f64(got[0]).reshape(n, -1), given), (f64(got[2]).reshape(n, top), tops)):
        assert np.array_equal(np.isnan(a), np.isnan(want)) and np.array_equal(np.isinf(a), np.isinf(want))
        ok = np.isfinite(want)
        far = np.where(ok, np.abs(np.where(ok, a, 0) - np.where(ok, want, 0)), 0)
        assert np.all(far <= room[:, None] + 5 * U * np.abs(np.where(ok, want, 0)))
    h = f64(got[1]).reshape(n)
    assert np.array_equal(np.isnan(h), np.isnan(entropy))
    ok = np.isfinite(entropy)
    room = room + U * ((2 * terms + 16) * d1 + 6 * d2 + 4 * d1 * d1)
    assert np.all(np.abs(h - entropy)[ok] <= room[ok])


def some_tokens(seed, rows, given, vocab, dev, dtype="int64"):
    import torch

    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, max(vocab, 1), (rows, given) if given else (rows,), generator=g).to(dtype_of(dtype)).to(dev)


VOCABS = [1, 2, 5, 7, 8, 9, 63, 100, 512, 1000, 2047, 2048, 2049, 4096, 4099, 8191, 20000, 32768, 50257, 131072]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_sizes(dev, dtype, vocab):
    import torch

    for rows, top, given in ((1, 20, 0), (3, 5, 2), (37, 1, 0)):
        x = logits_of(vocab + rows, rows, vocab, dtype, dev)
        tokens = some_tokens(rows, rows, given, vocab, dev)
        for kind in ("dense", "apart", "odd"):
            check(ph.token_log_probs(layouts(x, kind), tokens, top), x, tokens, top)
        heat = (0.3 + torch.rand(rows, generator=torch.Generator().manual_seed(vocab))).to(dev)
        mask = torch.rand((rows, vocab), generator=torch.Generator().manual_seed(vocab)).to(dev) < 0.3
        check(ph.token_log_probs(x, tokens, top, heat, layouts(mask, "odd")), x, tokens, top, heat, mask)
        check(ph.token_log_probs(x, tokens.int(), top, 0.7, mask[0]), x, tokens.int(), top, 0.7, mask[0])


@pytest.mark.parametrize("vocab", [40, 1000, 5000, 70000])
@pytest.mark.parametrize("top", [0, 1, 2, 33, 63, 64])
def test_tops(dev, vocab, top):
    """Rows in one piece and cut ones, up to as many alternatives as there are classes, more than there are places."""
    for rows in (2, 1100 if vocab <= 5000 else 3):
        x = logits_of(vocab, rows, vocab, "float32", dev)
        tokens = some_tokens(top, rows, 1, vocab, dev)
        check(ph.token_log_probs(x, tokens, top), x, tokens, top)


@pytest.mark.parametrize("vocab", [300, 3000, 20000, 131072])
def test_ties(dev, vocab):
    """Equal logits go by their places, however many there are; logits in step with the threads and in falling and
    rising order, which crowd the collected places."""
    import torch

    i = torch.arange(vocab, device=dev)
    rows = [torch.zeros(vocab, device=dev), -i.float(), i.float(), (i % 8 == 3).float(), (i // 8 % 64 == 5) * (i % 1000).float(),
            (i // 8 % 64 < 10).float() * 4 - (i % 7).float(), (i // 512 % 4 == 1) * (i % 3).float(),
            torch.where(i < vocab // 2, 1.0, 1.0 - 2.0 ** -20), torch.where(i % 2 == 0, 0.0, -0.0)]
    x = torch.stack([r.float() for r in rows])
    tokens = some_tokens(vocab, len(rows), 3, vocab, dev)
    for top in (1, 20, 64):
        for more in (1, 128):  # cut, and in one piece
            y = x.repeat(more, 1)
            got = ph.token_log_probs(y, tokens.repeat(more, 1), top)
            check([v[:len(rows)] for v in got], x, tokens, top)
            for v in got:
                assert torch.equal(v, v[:len(rows)].repeat(more, *([1] * (v.dim() - 1))))


def test_masks_that_crowd(dev):
    """Allowed places of a few classes only: more are collected than are kept at once."""
    import torch

    for vocab in (20000, 131072):
        i = torch.arange(vocab, device=dev)
        x = logits_of(vocab, 4, vocab, "bfloat16", dev)
        mask = torch.stack([i // 8 % 64 < 3, i % 512 == 0, i < 70, i >= vocab - 1])
        tokens = torch.stack([i[:1], i[:1], i[:1] + 69, i[-1:]])
        for top in (5, 64):
            for rows in (1, 300):
                got = ph.token_log_probs(x.repeat(rows, 1), tokens.repeat(rows, 1), top, 1.0, mask.repeat(rows, 1))
                check([v[:4] for v in got], x, tokens, top, 1.0, mask)


@pytest.mark.parametrize("vocab", [6, 100, 3000, 40000])
def test_edges(dev, vocab):
    """Nothing allowed, infinities and NaN in allowed and other places, temperatures of 0, infinity, negative and NaN,
    tokens outside the vocabulary."""
    import torch

    inf, nan = math.inf, math.nan
    x = logits_of(vocab, 16, vocab, "float32", dev)
    mask = torch.ones((16, vocab), dtype=torch.bool, device=dev)
    heat = torch.ones(16, device=dev)
    mask[0] = False
    x[1] = -inf
    x[2, 3] = nan
    x[3, 3], mask[3, 3] = nan, False
    x[4, 4] = inf
    x[5, 4], mask[5, 4] = inf, False
    x[6, :4] = -inf
    heat[7] = 0
    heat[8] = inf
    heat[9], x[9, 2] = inf, -inf
    heat[10] = -1
    heat[11] = nan
    heat[12], x[12, 5] = 0, inf
    heat[13], mask[13] = 0, False
    x[14, 0], x[14, 1], heat[14] = 3.4e38, -3.4e38, 5e37  # a difference past 32 bits
    heat[15] = 1e-40
    tokens = torch.tensor([[3, -1, vocab, 0, 5, 1, 4]] * 16, device=dev)
    for top in (0, 3, 8):
        for more in (1, 80):  # cut, and in one piece
            with np.errstate(all="ignore"):
                got = ph.token_log_probs(x.repeat(more, 1), tokens.repeat(more, 1), top, heat.repeat(more), mask.repeat(more, 1))
                check([v[-16:] for v in got], x, tokens, top, heat, mask)


def test_shapes(dev):
    import torch

    x = torch.randn((2, 3, 50), device=dev)
    t = torch.randint(0, 50, (2, 3), device=dev)
    check(ph.token_log_probs(x, t, 4), x, t, 4)
    check(ph.token_log_probs(x, t[..., None].expand(2, 3, 5).contiguous(), 4), x, t[..., None].expand(2, 3, 5), 4)
    a, h, b, c = ph.token_log_probs(x[0, 0], t[0, 0], 2)
    assert a.shape == () and h.shape == () and b.shape == (2,) and c.shape == (2,)
    a, h, b, c = ph.token_log_probs(x[0, 0], t[0], 0)
    assert a.shape == (3,) and b.shape == (0,) and c.shape == (0,)
    a, h, b, c = ph.token_log_probs(x[:0], t[:0], 2)
    assert a.shape == (0, 3) and h.shape == (0, 3) and b.shape == (0, 3, 2)
    a, h, b, c = ph.token_log_probs(x[..., :0], t, 2)  # no vocabulary
    assert (a == -math.inf).all() and (h == 0).all() and (b == -math.inf).all() and (c == -1).all()
    a, h, b, c = ph.token_log_probs(x, t.new_empty((2, 3, 0)), 2)
    assert a.shape == (2, 3, 0)


def test_against_probabilities(dev):
    """The sister operator's distribution, and a certain one: e^0 and no entropy."""
    import torch

    x = logits_of(5, 9, 5003, "bfloat16", dev)
    t = some_tokens(5, 9, 4, 5003, dev)
    p = ph.token_probabilities(x, 0.8)
    got = ph.token_log_probs(x, t, 10, 0.8)
    assert torch.allclose(got[0].exp(), p.gather(1, t), rtol=1e-4, atol=0)
    assert torch.allclose(got[2].exp(), p.gather(1, got[3]), rtol=1e-4, atol=0)
    one = torch.full((1, 3000), -math.inf, device=dev)
    one[0, 77] = 5.0
    a, h, b, c = ph.token_log_probs(one, torch.tensor([77], device=dev), 2)
    assert a.item() == 0 and h.item() == 0 and b.tolist() == [[0.0, -math.inf]] and c.tolist() == [[77, -1]]


def test_long_vocabulary(dev):
    """Places past 2^31 bytes; stretches that grow with the row."""
    import torch

    vocab = (1 << 29) + 5
    x = torch.full((2, vocab), -30.0, device=dev)
    x[0, -1], x[0, 7], x[1, 1 << 28], x[1, -3] = 5.0, 4.0, 6.0, 6.0
    t = torch.tensor([[vocab - 1, 7], [1 << 28, vocab - 3]], device=dev)
    a, h, b, c = ph.token_log_probs(x, t, 3)
    rest = (vocab - 2) * math.exp(-30)
    want = [[5 - math.log(math.exp(5) + math.exp(4) + rest), 4 - math.log(math.exp(5) + math.exp(4) + rest)],
            [6 - math.log(2 * math.exp(6) + rest)] * 2]
    assert c.tolist() == [[vocab - 1, 7, 0], [1 << 28, vocab - 3, 0]]
    assert np.allclose(f64(a), want, rtol=1e-5, atol=1e-5)

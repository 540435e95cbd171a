"""The operators in 8-bit floating point and the log probabilities as a program uses them: one after the other, on other
streams, captured into a graph and replayed, two at once, at the largest rows."""
import math

import numpy as np
import pytest

import fp8_reference as R
import pyPhantom as ph
from test_gpu_clear_ops import f64

pytestmark = pytest.mark.gpu

EPS = 1e-6


def model(dev, width, vocab, seed=3):
    """(gain, vocabulary's codes, scales, the vocabulary in 64 bits as the codes stand for it)."""
    import torch

    g = torch.Generator().manual_seed(seed)
    gain = (1 + 0.1 * torch.randn(width, generator=g)).to(dev)
    codes, scales = ph.quantize_fp8((torch.randn((vocab, width), generator=g) / width ** 0.5).to(dev), 128)
    real = codes.float().cpu().double().numpy() * R.spread(f64(scales), (vocab, width), 128)
    return gain, codes, scales, real


def step(states, residual, gain, codes, scales, tokens, top, heat, mask=None):
    import torch

    a, sa, total = ph.rms_norm_fp8(states, gain, EPS, residual)
    logits = ph.fp8_matmul(a, sa, codes, scales, None, torch.float32)
    return (a, sa, total, logits, *ph.token_log_probs(logits, tokens, top, heat, mask))


@pytest.mark.parametrize("rows,width,vocab", [(1, 256, 1000), (5, 4096, 20011), (40, 777, 5003)])
def test_chain(dev, rows, width, vocab):
    """Norm, vocabulary product, log probabilities: each step against the definition on what the step before gave, and
    the end against double precision."""
    import torch

    g = torch.Generator().manual_seed(rows)
    states, residual = (torch.randn((rows, width), generator=g).to(dev) for _ in range(2))
    gain, codes, scales, real = model(dev, width, vocab)
    tokens = torch.randint(0, vocab, (rows, 2), generator=g).to(dev)
    a, sa, total, logits, given, entropy, tops, places = step(states, residual, gain, codes, scales, tokens, 7, 0.9)
    # the product of the codes it was given: as test_gpu_fp8_ops.check_matmul
    values = a.float().cpu().double().numpy() * R.spread(f64(sa), (rows, width))
    want, size = values @ real.T, np.abs(values) @ np.abs(real).T
    assert np.all(np.abs(f64(logits) - want) <= 2 * (128 + sa.shape[1] + 12) * R.U * size + R.U * np.abs(want))
    ref = R.log_probs(f64(logits), tokens.cpu().numpy(), 7, np.full(rows, np.float32(0.9), np.float64))
    assert np.array_equal(places.cpu().numpy(), ref[3])
    # logits within +-10 at a temperature of 0.9: differences of two under 25, off by 2^-24 of themselves, a sum of up to
    # 20011 powers by 2^-21 of itself and the entropy by as much times 25; 10^-4 is 2^-13
    for got, w in ((given, ref[0]), (tops, ref[2]), (entropy, ref[1])):
        assert np.allclose(f64(got), w, rtol=0, atol=1e-4)
    # Against double precision from the states on: a code is off by 2^-4 of its value at most, independently, so a
    # logit, a sum of `width` products, by (2^-4 / sqrt(3)) (root of the sum of their squares) in the mean, and hardly any
    # by 6 times that.
    y = f64(states) + f64(residual)
    y = y / np.sqrt((y * y).mean(-1, keepdims=True) + EPS) * f64(gain)
    far = np.abs(f64(logits) - y @ real.T)
    assert np.all(far <= 6 * 2.0 ** -4 / 3 ** 0.5 * np.sqrt((y * y) @ (real * real).T) + 1e-4)


def test_answers_scored(dev):
    """Drafts checked and scored: the log probabilities of verify_drafts' own tokens, padding -infinity."""
    import torch

    g = torch.Generator().manual_seed(2)
    batch, drafts, vocab = 6, 4, 3001
    logits = (torch.randn((batch, drafts + 1, vocab), generator=g) * 3).to(dev)
    p = ph.token_probabilities(logits)
    x = torch.randint(0, vocab, (batch, drafts), generator=g).to(dev)
    x[:, 0] = logits[:, 0].argmax(-1)
    tokens, kept = ph.verify_drafts(x, p, torch.rand((batch, drafts), generator=g).to(dev),
                                    torch.empty((batch, vocab)).exponential_(generator=g).to(dev))
    given, entropy, _, places = ph.token_log_probs(logits, tokens, 1)
    assert given.shape == tokens.shape and torch.equal(torch.isinf(given), tokens < 0)
    there = tokens >= 0
    want = torch.log_softmax(logits.double(), -1).gather(-1, tokens.clamp(min=0)[..., None])[..., 0]
    assert torch.allclose(given[there].double(), want[there], rtol=0, atol=1e-5)
    assert torch.equal(places[..., 0], logits.argmax(-1))


def test_other_stream(dev):
    """Work queued behind slow work on a stream of its own, and on the default one in between."""
    import torch

    width, vocab = 512, 4000
    gain, codes, scales, _ = model(dev, width, vocab)
    x = torch.randn((9, width), device=dev)
    tokens = torch.arange(9, device=dev)
    want = step(x * 2, x, gain, codes, scales, tokens, 5, 1.0)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    slow = torch.randn((2048, 2048), device=dev)
    with torch.cuda.stream(s):
        for _ in range(20):
            slow = slow @ slow * 1e-3
        y = x * 2
        got = step(y, x, gain, codes, scales, tokens, 5, 1.0)
    step(x, x, gain, codes, scales, tokens, 5, 1.0)
    s.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a.float() if "float8" in str(a.dtype) else a, b.float() if "float8" in str(b.dtype) else b)


@pytest.mark.parametrize("rows,width,vocab,top", [(3, 512, 70001, 20), (300, 2048, 1000, 3), (70, 16384, 64, 0)])
def test_captured(dev, rows, width, vocab, top):
    """A graph of the whole step (workspaces, split sums, cut rows), replayed with other states and eager work between, and a
    second graph of the same step: every replay is the eager result."""
    import torch

    gain, codes, scales, _ = model(dev, width, vocab)
    x, r = torch.randn((rows, width), device=dev), torch.randn((rows, width), device=dev)
    tokens = torch.randint(0, vocab, (rows,), device=dev)
    heat = torch.rand(rows, device=dev) + 0.5
    mask = torch.rand((rows, vocab), device=dev) < 0.7

    def run():
        out = step(x, r, gain, codes, scales, tokens, top, heat, mask)
        narrow = ph.fp8_matmul(*out[:2], codes, scales, None, torch.bfloat16)
        return (*out, narrow)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        run()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    plain = lambda t: t.float() if "float8" in str(t.dtype) else t  # noqa: E731
    for turn in range(4):
        x.normal_()
        r.normal_()
        tokens.random_(0, vocab)
        want = [plain(t).clone() for t in run()]
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(want, out):
                assert torch.equal(a, plain(b)), turn
        if turn % 2:
            graphs[0][0].replay()  # one after the other without waiting
            graphs[1][0].replay()
            run()
            torch.cuda.synchronize()
            for graph, out in graphs:
                assert all(torch.equal(a, plain(b)) for a, b in zip(want, out))


def test_two_at_once(dev):
    """Split products and cut rows on two streams at the same time: workspaces are a call's own."""
    import torch

    from test_gpu_fp8_ops import operands

    sizes = [(128, 1000, 16384), (300, 1000, 12000)]
    args = [operands(i, *size, dev) for i, size in enumerate(sizes)]
    logits = [torch.randn((4, 131072), device=dev) for _ in range(2)]
    tokens = torch.zeros(4, dtype=torch.int64, device=dev)
    want = [(ph.fp8_matmul(*a), *ph.token_log_probs(x, tokens, 20)) for a, x in zip(args, logits)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = [None, None]
        for i in (0, 1, 0, 1):
            with torch.cuda.stream(streams[i]):
                got[i] = (ph.fp8_matmul(*args[i]), *ph.token_log_probs(logits[i], tokens, 20))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_crowded_rows(dev):
    """Rows whose largest logits stand in few classes, rising and falling: the threshold is found all the same."""
    import torch

    for vocab in (131072, 1 << 20):
        i = torch.arange(vocab, device=dev)
        few = (i // 8 % 64 < 3) & (i // 512 % 2 == 0)
        rising = torch.where(few, i.float(), -1e6)
        rows = torch.stack([rising, torch.where(few, -i.float(), -1e7), torch.where(few, 1.0, 0.0)])
        tokens = torch.zeros(3, dtype=torch.int64, device=dev)
        for more in (1, 20, 400) if vocab == 131072 else (1,):  # cut rows, long and ordinary workgroups
            _, _, tops, places = ph.token_log_probs(rows.repeat(more, 1), tokens.repeat(more), 64)
            order = torch.sort(rows, dim=-1, descending=True, stable=True).indices[:, :64]
            assert torch.equal(places, order.repeat(more, 1)) and not torch.isnan(tops).any()


def test_mask_and_logits_of_one_row(dev):
    """Logits and masks that are one row over and over, lengths of tokens past 32 bits, a mask that leaves a token."""
    import torch

    x = torch.randn(3000, device=dev)
    tokens = torch.tensor([5, 1 << 40, -(1 << 40), 2999, 1 << 32], device=dev)
    one = torch.zeros(3000, dtype=torch.bool, device=dev)
    one[2999] = True
    a = ph.token_log_probs(x.expand(5, 3000), tokens, 2, 1.0, one.expand(5, 3000))
    b = ph.token_log_probs(x.repeat(5, 1), tokens, 2, 1.0, one)
    for p, q in zip(a, b):
        assert torch.equal(p, q)
    assert a[0].tolist() == [-math.inf, -math.inf, -math.inf, 0.0, -math.inf]
    assert a[3].tolist() == [[2999, -1]] * 5 and a[1].tolist() == [0.0] * 5


def test_outputs_past_32_bits(dev):
    """More than 2^32 bytes of outputs: the last tile is where it belongs."""
    import torch

    m, n, k = 40000, 65537, 128
    a = torch.zeros((m, k), device=dev).to(torch.float8_e4m3fn)
    b = torch.zeros((n, k), device=dev).to(torch.float8_e4m3fn)
    one = torch.tensor(1.0, device=dev).to(torch.float8_e4m3fn)
    a.view(torch.uint8)[-1], b.view(torch.uint8)[-1] = one.view(torch.uint8), one.view(torch.uint8)
    a.view(torch.uint8)[0, 0], b.view(torch.uint8)[0, 0] = one.view(torch.uint8), one.view(torch.uint8)
    sa = torch.ones((m, 1), device=dev)
    sb = torch.ones((R.spans(n), 1), device=dev)
    out = ph.fp8_matmul(a, sa, b, sb, None, torch.bfloat16)
    assert out[0, 0] == 1 and out[-1, -1] == k and out[-1, 0] == 1 and out[0, -1] == 1
    assert int((out != 0).sum()) == 4


def test_most_columns(dev):
    """A token and as many columns as one launch without tiles forms, and one more; b has 2^33 bytes."""
    import torch

    k = 128
    one = torch.ones((1, k), device=dev).to(torch.float8_e4m3fn)
    sa = torch.full((1, 1), 2.0, device=dev)
    for n in ((1 << 26) - 1, 1 << 26):
        b = torch.zeros((n, k), dtype=torch.uint8, device=dev)
        b[-1], b[0], b[(1 << 25) + 5] = one.view(torch.uint8), one.view(torch.uint8), one.view(torch.uint8)
        sb = torch.ones((R.spans(n), 1), device=dev)
        sb[-1] = 3
        out = ph.fp8_matmul(one, sa, b.view(torch.float8_e4m3fn), sb, None, torch.float16)
        assert out[0, -1] == 6 * k and out[0, 0] == 2 * k and out[0, (1 << 25) + 5] == 2 * k
        assert int((out != 0).sum()) == 3
        del b, out


def test_example(dev):
    """examples/encrypted_decoding.py with the vocabulary in 8-bit floats runs, and says the tokens it kept."""
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "encrypted_decoding.py")
    spec = importlib.util.spec_from_file_location("encrypted_decoding", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    lines = []
    text, worst = module.run(rounds=2, say=lines.append, codes="e4m3")
    assert 2 <= len(text) <= 10 and all(0 <= t < 1000 for t in text) and len(lines) == 3
    # A code is off by 2^-4 of itself at most: a logit of deviation 1 by less than 2^-4 (both factors, independent, uniform
    # within their steps), probabilities by 2^-4 / 0.8 = 0.08 in the mean at most
    assert worst < 0.1
    with pytest.raises(ValueError):
        module.run(codes="fp4")

"""The clear operators in 8-bit floating point, and log probabilities, in numpy and 64 bits, from their definitions, for
the tests."""
import numpy as np

U = 2.0 ** -24  # one rounding to 32 bits, relative
SPAN = 128


def e4m3(q):
    """q to the nearest e4m3 number, ties to even, |q| <= 448: 4 significant bits, steps of 2^-9 below 2^-6."""
    q = np.asarray(q, np.float64)
    ulp = np.exp2(np.floor(np.log2(np.maximum(np.abs(q), 2.0 ** -6))) - 3)
    return np.rint(q / ulp) * ulp


def e4m3_step(q):
    """Distance of the e4m3 numbers around q."""
    return np.exp2(np.floor(np.log2(np.maximum(np.abs(q), 2.0 ** -6))) - 3)


def power_for(top):
    """The least power of two, 2^-126 or more, that takes `top` to 448 or less; 0 for 0, NaN for what is not finite."""
    top = np.asarray(top, np.float64)
    part, e = np.frexp(np.where(np.isfinite(top), top, 1.0))
    s = np.exp2(np.maximum(np.where(part > 0.875, e - 8, e - 9), -126).astype(np.float64))
    return np.where(np.isfinite(top), np.where(top > 0, s, 0.0), np.nan)


def spans(n):
    return -(-n // SPAN)


def block_tops(v, rows=1):
    """max|v| of blocks of `rows` x 128 of v [n, width]; NaN where a block has one, or an infinity."""
    n, width = v.shape
    whole = np.zeros((-(-n // rows) * rows, spans(width) * SPAN))
    whole[:n, :width] = np.where(np.isfinite(v), np.abs(v), np.nan)
    return whole.reshape(-1, rows, spans(width), SPAN).max((1, 3))


def spread(scales, shape, rows=1):
    """Scales of blocks, one for each element of a matrix of `shape`."""
    return np.repeat(np.repeat(scales, rows, 0), SPAN, 1)[:shape[0], :shape[1]]


def quantized(v, rows=1):
    """(codes as numbers, scales) of v [n, width]."""
    scales = power_for(block_tops(v, rows))
    each = spread(scales, v.shape, rows)
    with np.errstate(all="ignore"):
        codes = np.where(np.nan_to_num(each) > 0, e4m3(np.where(np.isfinite(v), v, 0) / each), 0.0)
    return codes, scales


def matmul(a, sa, b, sb, bias=None):
    """(product, sum of magnitudes, sum over eights of the largest products) of numbers a [m, k], b [n, k]."""
    m, k = a.shape
    n = b.shape[0]
    pad = spans(k) * SPAN - k
    A = np.pad(a, ((0, 0), (0, pad))) * np.repeat(sa, SPAN, 1)
    B = np.pad(b, ((0, 0), (0, pad))) * np.repeat(np.repeat(sb, SPAN, 0)[:n], SPAN, 1)
    out, size = A @ B.T, np.abs(A) @ np.abs(B).T
    # the matrix unit takes a number below 2^-6 for one of 2^-6 when it aligns products
    lift = np.repeat(np.abs(sa), SPAN, 1) * 2.0 ** -6, np.repeat(np.abs(np.repeat(sb, SPAN, 0)[:n]), SPAN, 1) * 2.0 ** -6
    E, F = np.maximum(np.abs(A), lift[0]), np.maximum(np.abs(B), lift[1])
    eights = np.zeros((m, n))
    for i in range(0, A.shape[1], 8):
        eights += (E[:, None, i:i + 8] * F[None, :, i:i + 8]).max(-1)
    return out + (0 if bias is None else bias), size, eights


def log_probs(logits, tokens, top, temperature, mask=None):
    """Rows [n, vocab], tokens [n, given], temperature [n]: (given, entropy, top values, top tokens, moments), moments
    [n, 3]: sum p |d|, sum p d^2, log of the sum of weights."""
    n, vocab = logits.shape
    given, entropy = np.full(tokens.shape, -np.inf), np.zeros(n)
    tops, places, moments = np.full((n, top), -np.inf), np.full((n, top), -1, np.int64), np.zeros((n, 3))
    for i in range(n):
        ok = np.ones(vocab, bool) if mask is None else (mask[i] if mask.ndim == 2 else mask)
        t, l = temperature[i], logits[i]
        v = l[ok]
        if v.size and (np.isnan(v).any() or not t >= 0 or (t > 0 and (v == np.inf).any())):
            lp = np.where(ok, np.nan, -np.inf)
            entropy[i] = np.nan
            tops[i] = np.nan
        else:
            if not v.size and not t >= 0:
                entropy[i] = np.nan
                tops[i] = np.nan
            lp = np.full(vocab, -np.inf)
            allowed = np.where(ok, l, -np.inf)
            order = np.argsort(-allowed, kind="stable")[:top]
            if v.size and v.max() > -np.inf:
                if t == 0:
                    lp[np.flatnonzero(ok)[v.argmax()]] = 0
                else:
                    with np.errstate(all="ignore"):
                        d = np.where(allowed > -np.inf, (allowed - v.max()) / t, -np.inf)
                    w = np.exp(d)
                    total = w.sum()
                    lp = d - np.log(total)
                    f = np.where(w > 0, d, 0)
                    entropy[i] = np.log(total) - (w * f).sum() / total
                    moments[i] = (w * -f).sum() / total, (w * f * f).sum() / total, np.log(total)
                there = allowed[order] > -np.inf
                tops[i, :order.size] = np.where(there, lp[order], -np.inf)
                places[i, :order.size] = np.where(there, order, -1)
        for j, x in enumerate(tokens[i]):
            if 0 <= x < vocab:
                given[i, j] = lp[x]
    return given, entropy, tops, places, moments

"""The clear operators in numpy and 64 bits, from their definitions, for the tests."""
import numpy as np

EPS = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # unit roundoff: 24, 8, 11 significant bits


def quantized(v):
    """(real-valued codes 127 v / max|v|, scales) of the rows of v; zero rows have 0 for both."""
    top = np.abs(v).max(-1) if v.shape[-1] else np.zeros(v.shape[:-1])
    with np.errstate(all="ignore"):
        return np.where(top[..., None] > 0, v / top[..., None] * 127, 0.0), top / 127


def rms_norm(x, weight, eps, residual=None):
    y = x if residual is None else x + residual
    return y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * weight


def probabilities(logits, temperature, mask=None):
    """Rows [n, vocab]; temperature [n]."""
    out = np.zeros(logits.shape)
    for i, (row, t) in enumerate(zip(logits, temperature)):
        ok = np.ones(row.shape, bool) if mask is None else mask[i] if mask.ndim == 2 else mask
        if not ok.any():
            continue
        v = row[ok]
        if np.isnan(v).any() or not t >= 0 or (t > 0 and (v == np.inf).any()):
            out[i, ok] = np.nan
        elif v.max() == -np.inf:
            pass
        elif t == 0:
            out[i, np.flatnonzero(ok)[v.argmax()]] = 1
        else:
            e = np.exp((v - v.max()) / t)
            out[i, ok] = e / e.sum()
    return out


def verify(drafts, p, u, e, q=None, lengths=None):
    """Lists of (tokens, accepted), one sequence after the other."""
    batch, places, vocab = p.shape
    tokens, accepted = np.full((batch, places), -1, np.int64), np.zeros(batch, np.int32)
    for b in range(batch):
        n, end = 0, places - 1 if lengths is None else min(max(int(lengths[b]), 0), places - 1)
        while n < end:
            x = drafts[b, n]
            if not 0 <= x < vocab or not u[b, n] * (1.0 if q is None else q[b, n, x]) < p[b, n, x]:
                break
            n += 1
        w = p[b, n]
        if n < end:
            if q is not None:
                less = w - q[b, n]
            else:
                less = w.copy()
                if 0 <= drafts[b, n] < vocab:
                    less[drafts[b, n]] = 0
            w = less if (less > 0).any() else w
        with np.errstate(all="ignore"):
            race = np.where(w > 0, w / e[b], 0.0)
        tokens[b, :n] = drafts[b, :n]
        tokens[b, n] = race.argmax() if vocab and (race > 0).any() else -1
        accepted[b] = n
    return tokens, accepted

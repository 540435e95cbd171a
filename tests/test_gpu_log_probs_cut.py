"""What rows may hold at their edges, in rows that are cut into stretches (few and long: two launches) and in the same
rows whole: infinities and NaN in allowed and other places, stretches that allow nothing, temperatures of 0, infinity,
negative, NaN and subnormal.  Against numpy in 64 bits, with test_gpu_log_probs.check's tolerances."""
import math

import numpy as np
import pytest

import pfa_native as P
import pyPhantom as ph
from test_gpu_log_probs import check, logits_of

pytestmark = pytest.mark.gpu

ROWS = 24
AT_ONCE = 12  # rows of a call: few enough to be cut at every one of these lengths


def edges(vocab, dev):
    """(logits, temperatures, mask): a kind of edge a row, the special places in the first, a middle and the last stretch."""
    import torch

    inf, nan = math.inf, math.nan
    mid, last = vocab // 2 + 3, vocab - 1
    x = logits_of(vocab, ROWS, vocab, "float32", dev)
    mask = torch.ones((ROWS, vocab), dtype=torch.bool, device=dev)
    heat = torch.ones(ROWS, device=dev)
    mask[0] = False
    x[1] = -inf
    x[2, mid] = nan
    x[3, mid], mask[3, mid] = nan, False
    x[4, last] = inf
    x[5, last], mask[5, last] = inf, False
    x[6, :mid] = -inf
    heat[7] = 0
    heat[8] = inf
    heat[9], x[9, mid:] = inf, -inf
    heat[10] = -1
    heat[11] = nan
    heat[12], x[12, mid], x[12, last] = 0, inf, inf
    heat[13], mask[13] = 0, False
    x[14, 0], x[14, last], heat[14] = 3.4e38, -3.4e38, 5e37  # a difference past 32 bits, brought back
    heat[15] = 1e-40
    mask[16, :last] = False
    mask[17, :vocab - 1000] = False
    heat[18], x[18, mid], x[18, last] = 0, 30.0, 30.0  # the lowest of two in different stretches
    heat[19], x[19] = 0, -inf
    x[20, mid], mask[20] = nan, False
    mask[20, mid] = True  # a NaN is all that is allowed
    x[21], x[21, mid] = -inf, 2.0
    heat[22] = 3e38
    x[23, :mid], x[23, mid:] = -3.4e38, 3.4e38  # a difference past 32 bits, of half a row
    return x, heat, mask


@pytest.mark.parametrize("vocab", [70000, 131072, 200003, 600000])
@pytest.mark.parametrize("top", [0, 3, 40])
def test_edges(dev, vocab, top):
    import torch

    assert all(P.log_probs_workspace(n, vocab) > 0 for n in range(1, AT_ONCE + 1))
    x, heat, mask = edges(vocab, dev)
    tokens = torch.tensor([[3, -1, vocab, 0, vocab - 1, vocab // 2 + 3, 1]] * ROWS, device=dev)
    with np.errstate(all="ignore"):
        for i in range(0, ROWS, AT_ONCE):
            part = slice(i, i + AT_ONCE)
            check(ph.token_log_probs(x[part], tokens[part], top, heat[part], mask[part]), x[part], tokens[part], top, heat[part],
                  mask[part])
        # the same rows whole
        more = vocab // 4096 // ROWS + 1
        assert P.log_probs_workspace(more * ROWS, vocab) == 0
        got = ph.token_log_probs(x.repeat(more, 1), tokens.repeat(more, 1), top, heat.repeat(more), mask.repeat(more, 1))
        check([v[-ROWS:] for v in got], x, tokens, top, heat, mask)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_edges_of_16_bits(dev, dtype):
    """One temperature for all rows, no mask: infinities and NaN in the logits themselves."""
    import torch

    vocab = 131072
    x = logits_of(9, 6, vocab, dtype, dev)
    x[0] = -math.inf
    x[1, vocab - 2] = math.nan
    x[2, 5] = math.inf
    x[3, 10:] = -math.inf
    x[4, :vocab - 3] = -math.inf
    tokens = torch.tensor([[vocab - 1, 2]] * 6, device=dev)
    assert P.log_probs_workspace(6, vocab) > 0
    with np.errstate(all="ignore"):
        for heat in (1.0, 0.0, 3.0):
            check(ph.token_log_probs(x, tokens, 12, heat), x, tokens, 12, heat)

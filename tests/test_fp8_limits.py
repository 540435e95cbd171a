"""The largest products that fp8_matmul forms, that all of its entry points refuse the same ones, and the arithmetic of
its 16-bit outputs (no GPU needed)."""
import ctypes as C

import numpy as np
import pytest

import pfa_native as P
from test_clear_ops import _abi
from test_gpu_fp8_precision import aligned_sum, power

MOST = 1 << 22  # tiles of a launch
KINDS = [0, 1, 2]
LARGEST = (1 << 31) - 1


def tiles(m, n, k, kind):
    rows, cols, splits = P.fp8_plan(m, n, k, kind)
    return -(-m // (rows or 16)) * -(-n // cols) * splits, (rows, cols, splits)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(1 << 28, 16, 16), (1 << 26, 300, 16), (1, 1 << 28, 16), (1, (1 << 30) - 256, 128),
                                   (16, 1 << 29, 128), (17, 1 << 28, 1), (200, 1 << 28, 256), ((1 << 30) - 256, 1, 1),
                                   (1 << 29, 128, 128), (1 << 18, 1 << 18, 64), (1 << 21, 65000, 130), (60, 1 << 28, 5)])
def test_large_products_have_a_plan(kind, m, n, k):
    """Where low tiles are too many for a launch, larger ones form the product, mostly empty ones if need be."""
    count, plan = tiles(m, n, k, kind)
    assert 0 < count < MOST, plan
    assert P.fp8_workspace(m, n, k, kind) == (4 * plan[2] * m * n if plan[2] > 1 else 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m,n,k", [(1, 1 << 30, 16), (LARGEST, 1, 1), (LARGEST, 60, 0), (LARGEST, 1000, 16), (LARGEST, LARGEST, 0), (1 << 20, 1 << 20, 130),
                                   (129, 1 << 30, 128)])
def test_larger_ones_are_refused(kind, m, n, k):
    """By the workspace's size, the plan and the product alike: no launch, no answer that the product does not keep."""
    p = 1 << 20  # an aligned address that nothing reads
    size = [C.c_size_t(0) for _ in range(3)]
    said = {_abi("pfa_fp8_workspace", m, n, k, kind, C.byref(size[0])),
            _abi("pfa_fp8_plan", m, n, k, kind, *(C.byref(v) for v in size)),
            _abi("pfa_fp8_matmul", p, k, p, 1, m, p, k, p, -(-k // 128), 1, None, m, n, k, p, kind, n, None, 0, None)}
    assert len(said) == 1, said
    (rc, words), = said
    assert rc == P.PFA_ERR_INVALID_ARGUMENT and "more outputs than one launch can form" in words


@pytest.mark.parametrize("kind", KINDS)
def test_rows_too_far_apart(kind):
    """Streamed rows have limits of their own, which the strides decide."""
    p, far = 1 << 20, (1 << 23) + 1
    for m, n, a_stride, b_stride in ((1048561, 16, far, 128), (2, 1 << 26, far, 128), (2, 1 << 26, 128, far)):
        rc, words = _abi("pfa_fp8_matmul", p, a_stride, p, 1, m, p, b_stride, p, 1, 1, None, m, n, 128, p, kind, n, None, 0,
                         None)
        assert rc == P.PFA_ERR_INVALID_ARGUMENT and "far apart" in words, words


def test_cut_is_no_more_than_stated():
    """Seven of eight products can lose less than 2^-13 of the largest product of powers each; with subnormal codes that is
    more than 2^-13 of the largest product itself."""
    rng = np.random.default_rng(4)
    worst = 0.0
    for _ in range(2000):
        a, b = (np.rint(rng.standard_normal(8) * 8) * np.exp2(rng.integers(-9, 6, 8)) for _ in range(2))
        at = np.where(a * b != 0, power(a) * power(b), 0.0).max()
        lost = abs(aligned_sum(a, b) - (a * b).sum())
        assert lost <= 7 * 2.0 ** -13 * at
        worst = max(worst, lost / (2.0 ** -13 * max(np.abs(a * b).max(), 1e-300)))
    assert worst > 1

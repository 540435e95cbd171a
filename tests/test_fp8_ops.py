"""What the operators in 8-bit floating point and the log probabilities refuse, in Python and at the C ABI (no GPU needed: a
refused call launches nothing), and the definitions in fp8_reference.py against closed forms and torch's conversion."""
import ctypes as C
import math
import re

import numpy as np
import pytest
import torch

import fp8_reference as R
import pfa_native as P
import pyPhantom as ph
from test_clear_ops import _abi, fake

F8, F32, BF16, I64, I32 = torch.float8_e4m3fn, torch.float32, torch.bfloat16, torch.int64, torch.int32


@pytest.mark.parametrize("call,word", [
    (lambda: ph.quantize_fp8(torch.zeros(2, 3)), "GPU"),
    (lambda: ph.quantize_fp8(fake(2, 3, dtype=torch.int8)), "float32"),
    (lambda: ph.quantize_fp8(fake(2, 3, dtype=torch.float64)), "float32"),
    (lambda: ph.quantize_fp8(fake(4, 6)[:, ::2]), "adjacent"),
    (lambda: ph.quantize_fp8(fake(20).as_strided((4, 5), (3, 1))), "overlap"),
    (lambda: ph.quantize_fp8(fake()), "dimension"),
    (lambda: ph.quantize_fp8(fake(2, 3), 64), "block_rows"),
    (lambda: ph.quantize_fp8(fake(2, 3), 1.0), "block_rows"),
    (lambda: ph.quantize_fp8(fake(2, 3, 4), 128), "two dimensions"),
    (lambda: ph.quantize_fp8(fake(4), 128), "two dimensions"),
    (lambda: ph.rms_norm_fp8(torch.zeros(2, 3), torch.zeros(3)), "GPU"),
    (lambda: ph.rms_norm_fp8(fake(2, 3), fake(4)), "weight"),
    (lambda: ph.rms_norm_fp8(fake(2, 3), fake(3, dtype=BF16)), "weight"),
    (lambda: ph.rms_norm_fp8(fake(2, 3), fake(3), -1e-6), "eps"),
    (lambda: ph.rms_norm_fp8(fake(2, 3), fake(3), math.inf), "eps"),
    (lambda: ph.rms_norm_fp8(fake(2, 3), fake(3), math.nan), "eps"),
    (lambda: ph.rms_norm_fp8(fake(2, 3), fake(3), 1e-6, fake(3, 3)), "residual"),
    (lambda: ph.rms_norm_fp8(fake(2, 3), fake(3), 1e-6, fake(2, 3, dtype=BF16)), "residual"),
    (lambda: ph.rms_norm_fp8(fake(2, 0), fake(0)), "empty"),
    (lambda: ph.fp8_matmul(torch.zeros(2, 3).to(F8), fake(2, 1), fake(4, 3, dtype=F8), fake(1, 1)), "GPU"),
    (lambda: ph.fp8_matmul(fake(2, 3), fake(2, 1), fake(4, 3, dtype=F8), fake(1, 1)), "float8_e4m3fn"),
    (lambda: ph.fp8_matmul(fake(2, 3, dtype=torch.float8_e5m2), fake(2, 1), fake(4, 3, dtype=F8), fake(1, 1)),
     "float8_e4m3fn"),
    (lambda: ph.fp8_matmul(fake(2, 3, dtype=F8), fake(2, 1), fake(4, 5, dtype=F8), fake(1, 1)), "multiply"),
    (lambda: ph.fp8_matmul(fake(2, 3, dtype=F8), fake(2, 1), fake(1, 4, 3, dtype=F8), fake(1, 1)), "multiply"),
    (lambda: ph.fp8_matmul(fake(2, 3, dtype=F8), fake(3, 1), fake(4, 3, dtype=F8), fake(1, 1)), "a_scales"),
    (lambda: ph.fp8_matmul(fake(2, 3, dtype=F8), fake(2, 2), fake(4, 3, dtype=F8), fake(1, 1)), "a_scales"),
    (lambda: ph.fp8_matmul(fake(2, 3, dtype=F8), fake(2), fake(4, 3, dtype=F8), fake(1, 1)), "a_scales"),
    (lambda: ph.fp8_matmul(fake(2, 3, dtype=F8), fake(2, 1, dtype=BF16), fake(4, 3, dtype=F8), fake(1, 1)), "a_scales"),
    (lambda: ph.fp8_matmul(fake(2, 3, dtype=F8), fake(2, 1), fake(4, 3, dtype=F8), fake(4, 1)), "b_scales"),
    (lambda: ph.fp8_matmul(fake(2, 3, dtype=F8), fake(2, 1), fake(130, 3, dtype=F8), fake(1, 1)), "b_scales"),
    (lambda: ph.fp8_matmul(fake(2, 300, dtype=F8), fake(2, 3), fake(4, 300, dtype=F8), fake(1, 2)), "b_scales"),
    (lambda: ph.fp8_matmul(fake(2, 3, dtype=F8), fake(2, 1), fake(4, 3, dtype=F8), fake(1, 1), fake(3)), "bias"),
    (lambda: ph.fp8_matmul(fake(2, 3, dtype=F8), fake(2, 1), fake(4, 3, dtype=F8), fake(1, 1), None, F8), "out_dtype"),
    (lambda: ph.fp8_matmul(fake(2, 3, dtype=F8), fake(2, 1), fake(3, 4, dtype=F8).t(), fake(1, 1)), "adjacent"),
    (lambda: ph.token_log_probs(torch.zeros(2, 3), torch.zeros(2, dtype=I64)), "GPU"),
    (lambda: ph.token_log_probs(fake(2, 3, dtype=I64), fake(2, dtype=I64)), "float32"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(2)), "tokens"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(3, dtype=I64)), "tokens"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(3, 2, dtype=I64)), "tokens"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(2, 1, 1, dtype=I64)), "tokens"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(4, 2, dtype=I64).t()), "tokens"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(4, dtype=I64)[::2]), "contiguous"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(2, dtype=I64), 65), "top"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(2, dtype=I64), -1), "top"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(2, dtype=I64), 1.0), "top"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(2, dtype=I64), 1, -0.5), "temperature"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(2, dtype=I64), 1, math.inf), "temperature"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(2, dtype=I64), 1, fake(3)), "temperature"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(2, dtype=I64), 1, 1.0, fake(2, 3)), "mask"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(2, dtype=I64), 1, 1.0, fake(2, dtype=torch.bool)), "mask"),
    (lambda: ph.token_log_probs(fake(2, 3), fake(2, dtype=I64), 1, 1.0, fake(6, dtype=torch.bool)[::2]), "adjacent"),
    (lambda: ph.token_log_probs(fake(4, 6)[:, ::2], fake(4, dtype=I64)), "adjacent"),
])
def test_refusals(call, word):
    with pytest.raises(ValueError, match=word):
        call()


def test_abi_refusals():
    """Null pointers, unknown types, sizes and strides out of range, misaligned tensors: INVALID_ARGUMENT, no launch."""
    buf = C.create_string_buffer(4096)
    p = (C.addressof(buf) + 63) & ~63
    big = 1 << 31
    cases = [
        ("pfa_quantize_fp8", (p, 8, 3, 1, 8, 1, p, 8, p, 1, 1, None), "type"),
        ("pfa_quantize_fp8", (p, 8, 0, 1, 8, 2, p, 8, p, 1, 1, None), "1 or 128"),
        ("pfa_quantize_fp8", (None, 8, 0, 1, 8, 1, p, 8, p, 1, 1, None), "null"),
        ("pfa_quantize_fp8", (p, 4, 0, 2, 8, 1, p, 8, p, 1, 1, None), "overlap"),
        ("pfa_quantize_fp8", (p, 8, 0, 2, 8, 1, p, 0, p, 1, 1, None), "overlap"),
        ("pfa_quantize_fp8", (p, 8, 0, 2, 8, 1, p, 8, p, 0, 1, None), "scales overlap"),
        ("pfa_quantize_fp8", (p, 200, 0, 1, 200, 1, p, 200, p, 1, 0, None), "scales overlap"),
        ("pfa_quantize_fp8", (p + 1, 8, 0, 1, 8, 1, p, 8, p, 1, 1, None), "aligned"),
        ("pfa_quantize_fp8", (p, 8, 0, 1, 8, 1, p, 8, p + 2, 1, 1, None), "aligned"),
        ("pfa_quantize_fp8", (p, 8, 0, big, 8, 1, p, 8, p, 1, 1, None), "rows"),
        ("pfa_quantize_fp8", (p, big, 0, 1, (1 << 30) + 1, 1, p, big, p, 1, 1, None), "2\\^30"),
        ("pfa_rms_norm_fp8", (p, 8, None, 0, None, 0, 1, 8, 1e-6, None, 0, p, 8, p, 1, 1, None), "null"),
        ("pfa_rms_norm_fp8", (p, 8, p, 8, p, 0, 1, 8, 1e-6, None, 0, p, 8, p, 1, 1, None), "null"),
        ("pfa_rms_norm_fp8", (p, 8, None, 0, p, 0, 1, 8, -1.0, None, 0, p, 8, p, 1, 1, None), "eps"),
        ("pfa_rms_norm_fp8", (p, 8, None, 0, p, 0, 1, 8, math.inf, None, 0, p, 8, p, 1, 1, None), "eps"),
        ("pfa_rms_norm_fp8", (p, 8, None, 0, p, 0, 1, 0, 1e-6, None, 0, p, 8, p, 1, 1, None), "empty"),
        ("pfa_rms_norm_fp8", (p, 8, None, 0, p + 1, 1, 1, 8, 1e-6, None, 0, p, 8, p, 1, 1, None), "aligned"),
        ("pfa_rms_norm_fp8", (p, 8, None, 0, p, 0, 2, 8, 1e-6, None, 0, p, 8, p, 0, 1, None), "scales overlap"),
        ("pfa_fp8_matmul", (p, 8, None, 1, 1, p, 8, p, 1, 1, None, 1, 1, 8, p, 0, 1, None, 0, None), "null"),
        ("pfa_fp8_matmul", (p, 8, p, 1, 1, p, 4, p, 1, 1, None, 1, 2, 8, p, 0, 2, None, 0, None), "overlap"),
        ("pfa_fp8_matmul", (p, 8, p, 1, 1, p, 8, p, 1, 1, None, 2, 2, 8, p, 0, 1, None, 0, None), "overlap"),
        ("pfa_fp8_matmul", (p, 8, p, 1, 1, p, 8, p, 1, 1, None, 1, 1, 8, p, 9, 1, None, 0, None), "type"),
        ("pfa_fp8_matmul", (p, 8, p, 1, 1, p, 8, p, 1, 1, None, 1, 1, 8, p + 1, 1, 1, None, 0, None), "aligned"),
        ("pfa_fp8_matmul", (p, 8, p + 2, 1, 1, p, 8, p, 1, 1, None, 1, 1, 8, p, 1, 1, None, 0, None), "aligned"),
        ("pfa_fp8_matmul", (p, 8, p, 1, 1, p, 8, p, 1, 1, None, 1, 1, 8, p, 1, 1, None, 64, None), "workspace"),
        ("pfa_fp8_matmul", (p, 8, p, 1, 1, p, 8, p, 1, 1, None, 1, 1, 8, p, 1, 1, p + 8, 64, None), "workspace"),
        ("pfa_fp8_matmul", (p, big, p, 1, 1, p, big, p, 1, 1, None, 1, 1, big, p, 1, 1, None, 0, None), "2\\^31"),
        ("pfa_fp8_workspace", (1, 1, 1, 0, None), "null"),
        ("pfa_fp8_workspace", (1, 1, 1, 5, C.pointer(C.c_size_t(0))), "type"),
        ("pfa_log_probs_workspace", (1, 1, None), "null"),
        ("pfa_token_log_probs", (p, 8, 0, 1, 8, p, 4, 1, 1, None, -1.0, None, 0, p, p, p, p, None, 0, None), "temperature"),
        ("pfa_token_log_probs", (p, 8, 0, 1, 8, p, 4, 1, 1, None, math.nan, None, 0, p, p, p, p, None, 0, None),
         "temperature"),
        ("pfa_token_log_probs", (p, 8, 7, 1, 8, p, 4, 1, 1, None, 1.0, None, 0, p, p, p, p, None, 0, None), "type"),
        ("pfa_token_log_probs", (p, 8, 0, 1, 8, p, 2, 1, 1, None, 1.0, None, 0, p, p, p, p, None, 0, None), "bytes"),
        ("pfa_token_log_probs", (p, 8, 0, 1, 8, p, 4, 1, 65, None, 1.0, None, 0, p, p, p, p, None, 0, None), "64"),
        ("pfa_token_log_probs", (p, 4, 0, 2, 8, p, 4, 1, 1, None, 1.0, None, 0, p, p, p, p, None, 0, None), "overlap"),
        ("pfa_token_log_probs", (p, 8, 0, 2, 8, p, 4, 1, 1, None, 1.0, p, 4, p, p, p, p, None, 0, None), "overlap"),
        ("pfa_token_log_probs", (None, 8, 0, 1, 8, p, 4, 1, 1, None, 1.0, None, 0, p, p, p, p, None, 0, None), "null"),
        ("pfa_token_log_probs", (p, 8, 0, 1, 8, None, 4, 1, 1, None, 1.0, None, 0, p, p, p, p, None, 0, None), "null"),
        ("pfa_token_log_probs", (p, 8, 0, 1, 8, p, 4, 1, 1, None, 1.0, None, 0, p, p, p, None, None, 0, None), "null"),
        ("pfa_token_log_probs", (p, 8, 0, 1, 8, p + 4, 8, 1, 1, None, 1.0, None, 0, p, p, p, p, None, 0, None), "aligned"),
        ("pfa_token_log_probs", (p, 1 << 17, 0, 1, 1 << 17, p, 4, 1, 1, None, 1.0, None, 0, p, p, p, p, None, 0, None),
         "workspace"),
    ]
    for name, args, word in cases:
        rc, said = _abi(name, *args)
        assert rc == P.PFA_ERR_INVALID_ARGUMENT and re.search(word, said), (name, args, rc, said)


def test_abi_empty_calls_launch_nothing():
    ok = P.PFA_OK
    assert _abi("pfa_quantize_fp8", None, 0, 0, 0, 8, 1, None, 0, None, 0, 0, None)[0] == ok
    assert _abi("pfa_quantize_fp8", None, 0, 0, 8, 0, 128, None, 0, None, 0, 0, None)[0] == ok
    assert _abi("pfa_rms_norm_fp8", None, 0, None, 0, None, 1, 0, 8, 0.0, None, 0, None, 0, None, 0, 0, None)[0] == ok
    assert _abi("pfa_fp8_matmul", None, 0, None, 0, 0, None, 0, None, 0, 0, None, 0, 5, 5, None, 0, 0, None, 0, None)[0] == ok
    assert _abi("pfa_token_log_probs", None, 0, 0, 0, 5, None, 4, 1, 1, None, 1.0, None, 0, None, None, None, None, None, 0,
                None)[0] == ok


def test_workspace_sizes():
    """Rows that are cut need room for their stretches, as many as rows; many rows need none."""
    assert P.log_probs_workspace(1, 131072) > 0 and P.log_probs_workspace(4096, 131072) == 0
    assert P.log_probs_workspace(5, 131072) % 5 == 0 and P.log_probs_workspace(3, 1000) == 0
    assert P.log_probs_workspace(1, 1 << 30) <= 256 * 32  # stretches grow with the row


# ------------------------------------------------------------- the definitions
def test_reference_numbers():
    """The reference's rounding is torch's conversion, at every code, every tie and beside it; powers at the borders."""
    c = torch.arange(256, dtype=torch.uint8).view(F8).float()
    c = c[c.isfinite()].unique()
    ties = (c[1:] + c[:-1]) / 2
    x = torch.cat([c, ties, torch.nextafter(ties, ties + 1), torch.nextafter(ties, ties - 1),
                   torch.linspace(-448, 448, 9001), torch.linspace(-0.05, 0.05, 9001)])
    assert np.array_equal(R.e4m3(x.double().numpy()), x.to(F8).float().double().numpy())
    tops = [0.0, 448.0, np.nextafter(448, 500), 224.0, 1.0, 1e-45, 2.0 ** -118 * 1.75, 3.4028234663852886e38]
    assert np.array_equal(R.power_for(tops), [0, 1, 2, 0.5, 2.0 ** -8, 2.0 ** -126, 2.0 ** -126, 2.0 ** 120])
    assert np.isnan(R.power_for([np.nan, np.inf])).all()


def test_reference_blocks():
    v = np.zeros((3, 130))
    v[0, 0], v[1, 129], v[2, 5] = 896.0, -1.0, 30.0
    codes, scales = R.quantized(v)
    assert scales.tolist() == [[2.0, 0.0], [0.0, 2.0 ** -8], [0.125, 0.0]]
    assert codes[0, 0] == 448 and codes[1, 129] == -256 and codes[2, 5] == 240
    codes, scales = R.quantized(v, 128)
    assert scales.tolist() == [[2.0, 2.0 ** -8]] and codes[2, 5] == 15
    out, size, _ = R.matmul(np.ones((2, 130)), np.array([[2.0, 3.0], [1.0, 0.0]]), -np.ones((129, 130)),
                            np.array([[1.0, 10.0], [0.5, 0.0]]), np.zeros(129))
    assert out[:, 0].tolist() == [-316, -128] and out[:, 128].tolist() == [-128, -64] and size[0, 0] == 316


def test_reference_log_probs():
    x = np.log(np.array([[1.0, 2.0, 5.0, 2.0]]))
    given, entropy, tops, places, _ = R.log_probs(x, np.array([[2, 0, 7]]), 3, np.array([1.0]))
    p = np.array([0.1, 0.2, 0.5, 0.2])
    assert np.allclose(given, [[np.log(0.5), np.log(0.1), -np.inf]]) and np.allclose(entropy, -(p * np.log(p)).sum())
    assert places.tolist() == [[2, 1, 3]] and np.allclose(tops, np.log([[0.5, 0.2, 0.2]]))
    given, entropy, tops, places, _ = R.log_probs(x, np.array([[2, 0]]), 2, np.array([0.0]), np.array([True, True, False, True]))
    assert given.tolist() == [[-np.inf, -np.inf]] and entropy[0] == 0 and places.tolist() == [[1, 3]]
    assert tops.tolist() == [[0, -np.inf]]

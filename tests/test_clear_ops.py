"""What the clear operators refuse, in Python and at the C ABI (no GPU needed: a refused call
launches nothing), and the definitions in clear_reference.py against closed forms."""
import ctypes as C

import numpy as np
import pytest
import torch

import clear_reference as R
import pfa_native as P
import pyPhantom as ph


def test_public_names():
    import clear_ops

    assert sorted(clear_ops.__all__) == sorted(ph._CLEAR_OPS)
    for name in ph._CLEAR_OPS:
        assert getattr(ph, name) is getattr(clear_ops, name) and getattr(ph, name).__doc__
    with pytest.raises(AttributeError):
        ph.no_such_operator


class Fake(torch.Tensor):
    """A tensor that says it is on a GPU: what is refused is refused before its memory matters."""

    @property
    def is_cuda(self):
        return True


def fake(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(Fake)


I8, F32, BF16, I64 = torch.int8, torch.float32, torch.bfloat16, torch.int64


@pytest.mark.parametrize("call,word", [
    (lambda: ph.quantize_int8(torch.zeros(2, 3)), "GPU"),
    (lambda: ph.quantize_int8(fake(2, 3, dtype=I8)), "float32"),
    (lambda: ph.quantize_int8(fake(2, 3, dtype=torch.float64)), "float32"),
    (lambda: ph.quantize_int8(fake(4, 6)[:, ::2]), "adjacent"),
    (lambda: ph.quantize_int8(fake(4, 6).t()), "adjacent"),
    (lambda: ph.quantize_int8(fake(20).as_strided((4, 5), (3, 1))), "overlap"),
    (lambda: ph.quantize_int8(fake()), "dimension"),
    (lambda: ph.rms_norm_int8(torch.zeros(2, 3), torch.zeros(3)), "GPU"),
    (lambda: ph.rms_norm_int8(fake(2, 3), fake(4)), "weight"),
    (lambda: ph.rms_norm_int8(fake(2, 3), fake(3, dtype=BF16)), "weight"),
    (lambda: ph.rms_norm_int8(fake(2, 3), fake(6)[::2]), "weight"),
    (lambda: ph.rms_norm_int8(fake(2, 3), fake(3), -1e-6), "eps"),
    (lambda: ph.rms_norm_int8(fake(2, 3), fake(3), float("nan")), "eps"),
    (lambda: ph.rms_norm_int8(fake(2, 3), fake(3), 1e-6, fake(3, 3)), "residual"),
    (lambda: ph.rms_norm_int8(fake(2, 3), fake(3), 1e-6, fake(2, 3, dtype=BF16)), "residual"),
    (lambda: ph.rms_norm_int8(fake(2, 0), fake(0)), "empty"),
    (lambda: ph.int8_matmul(fake(2, 3), fake(2), fake(4, 3, dtype=I8), fake(4)), "int8"),
    (lambda: ph.int8_matmul(fake(2, 3, dtype=I8), fake(2), fake(4, 5, dtype=I8), fake(4)), "multiply"),
    (lambda: ph.int8_matmul(fake(2, 3, dtype=I8), fake(3), fake(4, 3, dtype=I8), fake(4)), "a_scales"),
    (lambda: ph.int8_matmul(fake(2, 3, dtype=I8), fake(2), fake(4, 3, dtype=I8), fake(5)), "b_scales"),
    (lambda: ph.int8_matmul(fake(2, 3, dtype=I8), fake(2, dtype=BF16), fake(4, 3, dtype=I8), fake(4)), "a_scales"),
    (lambda: ph.int8_matmul(fake(2, 3, dtype=I8), fake(2), fake(4, 3, dtype=I8), fake(4), fake(3)), "bias"),
    (lambda: ph.int8_matmul(fake(2, 3, dtype=I8), fake(2), fake(4, 3, dtype=I8), fake(4), None, I8), "out_dtype"),
    (lambda: ph.int8_matmul(fake(2, 3, dtype=I8), fake(2), fake(3, 4, dtype=I8).t(), fake(4)), "adjacent"),
    (lambda: ph.int8_matmul(fake(2, 3, dtype=I8), fake(2), fake(1, 4, 3, dtype=I8), fake(4)), "multiply"),
    (lambda: ph.token_probabilities(torch.zeros(2, 3)), "GPU"),
    (lambda: ph.token_probabilities(fake(2, 3, dtype=I64)), "float32"),
    (lambda: ph.token_probabilities(fake(2, 3), -0.5), "temperature"),
    (lambda: ph.token_probabilities(fake(2, 3), float("inf")), "temperature"),
    (lambda: ph.token_probabilities(fake(2, 3), fake(3)), "temperature"),
    (lambda: ph.token_probabilities(fake(2, 3), fake(2, dtype=BF16)), "temperature"),
    (lambda: ph.token_probabilities(fake(2, 3), 1.0, fake(2, 3)), "mask"),
    (lambda: ph.token_probabilities(fake(2, 3), 1.0, fake(2, dtype=torch.bool)), "mask"),
    (lambda: ph.token_probabilities(fake(2, 3), 1.0, fake(6, dtype=torch.bool)[::2]), "adjacent"),
    (lambda: ph.verify_drafts(fake(2, 1, dtype=I64), torch.zeros(2, 2, 5), fake(2, 1), fake(2, 5)), "GPU"),
    (lambda: ph.verify_drafts(fake(2, 1), fake(2, 2, 5), fake(2, 1), fake(2, 5)), "draft_tokens"),
    (lambda: ph.verify_drafts(fake(2, 2, dtype=I64), fake(2, 2, 5), fake(2, 1), fake(2, 5)), "draft_tokens"),
    (lambda: ph.verify_drafts(fake(2, 1, dtype=I64), fake(2, 0, 5), fake(2, 1), fake(2, 5)), "target_probs"),
    (lambda: ph.verify_drafts(fake(2, 1, dtype=I64), fake(2, 5), fake(2, 1), fake(2, 5)), "target_probs"),
    (lambda: ph.verify_drafts(fake(2, 1, dtype=I64), fake(2, 2, 5), fake(2, 2), fake(2, 5)), "uniforms"),
    (lambda: ph.verify_drafts(fake(2, 1, dtype=I64), fake(2, 2, 5), fake(2, 1), fake(2, 4)), "noise"),
    (lambda: ph.verify_drafts(fake(2, 1, dtype=I64), fake(2, 2, 5), fake(2, 1), fake(2, 5), fake(2, 2, 5)),
     "draft_probs"),
    (lambda: ph.verify_drafts(fake(2, 1, dtype=I64), fake(2, 2, 5), fake(2, 1), fake(2, 5), fake(2, 1, 5, dtype=BF16)),
     "draft_probs"),
    (lambda: ph.verify_drafts(fake(2, 1, dtype=I64), fake(2, 2, 5), fake(2, 1), fake(2, 5), None, fake(2)), "lengths"),
    (lambda: ph.verify_drafts(fake(2, 1, dtype=I64), fake(2, 5, 2).transpose(1, 2), fake(2, 1), fake(2, 5)),
     "adjacent"),
])
def test_refusals(call, word):
    with pytest.raises(ValueError, match=word):
        call()


def _abi(name, *args):
    rc = getattr(P.lib(), name)(*args)
    return rc, P.lib().pfa_last_error().decode()


def test_abi_refusals():
    """Null pointers, unknown types, sizes and strides out of range, misaligned tensors: INVALID_ARGUMENT, no launch."""
    bad = P.PFA_ERR_INVALID_ARGUMENT
    buf = C.create_string_buffer(4096)
    p = (C.addressof(buf) + 63) & ~63
    cases = [
        ("pfa_quantize_int8", (p, 8, 3, 1, 8, p, 8, p, None), "type"),
        ("pfa_quantize_int8", (None, 8, 0, 1, 8, p, 8, p, None), "null"),
        ("pfa_quantize_int8", (p, 4, 0, 2, 8, p, 8, p, None), "overlap"),
        ("pfa_quantize_int8", (p, 8, 0, 2, 8, p, 0, p, None), "overlap"),
        ("pfa_quantize_int8", (p + 1, 8, 0, 1, 8, p, 8, p, None), "aligned"),
        ("pfa_quantize_int8", (p, 8, 0, 1 << 31, 8, p, 8, p, None), "rows"),
        ("pfa_quantize_int8", (p, 1 << 31, 0, 1, (1 << 30) + 1, p, 1 << 31, p, None), "2\\^30"),
        ("pfa_rms_norm_int8", (p, 8, None, 0, None, 0, 1, 8, 1e-6, None, 0, p, 8, p, None), "null"),
        ("pfa_rms_norm_int8", (p, 8, p, 8, p, 0, 1, 8, 1e-6, None, 0, p, 8, p, None), "null"),
        ("pfa_rms_norm_int8", (p, 8, None, 0, p, 0, 1, 8, -1.0, None, 0, p, 8, p, None), "eps"),
        ("pfa_rms_norm_int8", (p, 8, None, 0, p, 0, 1, 0, 1e-6, None, 0, p, 8, p, None), "empty"),
        ("pfa_rms_norm_int8", (p, 8, None, 0, p + 1, 1, 1, 8, 1e-6, None, 0, p, 8, p, None), "aligned"),
        ("pfa_int8_matmul", (p, 131072, p, p, 131072, p, None, 1, 1, 131072, p, 0, 1, None, 0, None), "131071"),
        ("pfa_int8_matmul", (p, 8, None, p, 8, p, None, 1, 1, 8, p, 0, 1, None, 0, None), "null"),
        ("pfa_int8_matmul", (p, 8, p, p, 4, p, None, 1, 2, 8, p, 0, 2, None, 0, None), "overlap"),
        ("pfa_int8_matmul", (p, 8, p, p, 8, p, None, 2, 2, 8, p, 0, 1, None, 0, None), "overlap"),
        ("pfa_int8_matmul", (p, 8, p, p, 8, p, None, 1, 1, 8, p, 9, 1, None, 0, None), "type"),
        ("pfa_int8_matmul", (p, 8, p, p, 8, p, None, 1, 1, 8, p + 1, 1, 1, None, 0, None), "aligned"),
        ("pfa_int8_matmul", (p, 8, p, p, 8, p, None, 1, 1, 8, p, 1, 1, None, 64, None), "workspace"),
        ("pfa_token_probabilities", (p, 8, 0, 1, 8, None, -1.0, None, 0, p, None, 0, None), "temperature"),
        ("pfa_token_probabilities", (p, 8, 7, 1, 8, None, 1.0, None, 0, p, None, 0, None), "type"),
        ("pfa_token_probabilities", (p, 4, 0, 2, 8, None, 1.0, None, 0, p, None, 0, None), "overlap"),
        ("pfa_token_probabilities", (p, 8, 0, 2, 8, None, 1.0, p, 4, p, None, 0, None), "overlap"),
        ("pfa_token_probabilities", (p, 1 << 17, 0, 4, 1 << 17, None, 1.0, None, 0, p, None, 0, None), "workspace"),
        ("pfa_verify_drafts", (p, 8, None, 4, 1, 1, 1 << 17, p, 1 << 18, 1 << 17, None, 0, 0, 0, p, p, 8, p, p, None, 0,
                               None), "workspace"),
        ("pfa_int8_matmul", (p, 16384, p, p, 16384, p, None, 64, 64, 16384, p, 0, 64, None, 0, None), "workspace"),
        ("pfa_token_probabilities", (None, 8, 0, 1, 8, None, 1.0, None, 0, p, None, 0, None), "null"),
        ("pfa_verify_drafts", (p, 2, None, 4, 1, 1, 8, p, 16, 8, None, 0, 0, 0, p, p, 8, p, p, None, 0, None), "bytes"),
        ("pfa_verify_drafts", (p, 8, p, 3, 1, 1, 8, p, 16, 8, None, 0, 0, 0, p, p, 8, p, p, None, 0, None), "bytes"),
        ("pfa_verify_drafts", (p, 8, None, 4, 1, 1, 8, None, 16, 8, None, 0, 0, 0, p, p, 8, p, p, None, 0, None), "null"),
        ("pfa_verify_drafts", (p, 8, None, 4, 1, 1, 8, p + 2, 16, 8, None, 0, 0, 0, p, p, 8, p, p, None, 0, None),
         "aligned"),
    ]
    import re

    for name, args, word in cases:
        rc, said = _abi(name, *args)
        assert rc == bad and re.search(word, said), (name, args, rc, said)


def test_abi_empty_calls_launch_nothing():
    assert _abi("pfa_quantize_int8", None, 0, 0, 0, 8, None, 0, None, None)[0] == P.PFA_OK
    assert _abi("pfa_rms_norm_int8", None, 0, None, 0, None, 1, 0, 8, 0.0, None, 0, None, 0, None, None)[0] == P.PFA_OK
    assert _abi("pfa_int8_matmul", None, 0, None, None, 0, None, None, 0, 5, 5, None, 0, 0, None, 0, None)[0] == P.PFA_OK
    assert _abi("pfa_token_probabilities", None, 0, 0, 0, 5, None, 1.0, None, 0, None, None, 0, None)[0] == P.PFA_OK
    assert _abi("pfa_verify_drafts", None, 8, None, 4, 0, 0, 5, None, 0, 0, None, 0, 0, 0, None, None, 0, None, None,
                None, 0, None)[0] == P.PFA_OK


def test_workspace_sizes():
    """What the calls need is what the queries say; short rows and large products need nothing."""
    assert P.token_workspace(5, 131072) > 0 and P.token_workspace(1000, 8192) == 0
    assert P.matmul_workspace(64, 64, 16384) % (64 * 64 * 4) == 0 and P.matmul_workspace(64, 64, 16384) > 0
    assert P.matmul_workspace(4096, 16384, 4096) == 0 and P.matmul_workspace(1, 4096, 16384) == 0
    for name, args in (("pfa_token_workspace", (1, 1)), ("pfa_matmul_workspace", (1, 1, 1))):
        assert _abi(name, *args, None)[0] == P.PFA_ERR_INVALID_ARGUMENT
    with pytest.raises(ValueError, match="131071"):
        P.matmul_workspace(1, 1, 131072)


def test_reference_closed_forms():
    real, scale = R.quantized(np.array([[1.0, -2.0, 0.5], [0.0, 0.0, 0.0]]))
    assert np.allclose(real, [[63.5, -127, 31.75], [0, 0, 0]]) and np.allclose(scale, [2 / 127, 0])
    v = R.rms_norm(np.array([[3.0, 4.0]]), np.array([1.0, 2.0]), 0.0)
    assert np.allclose(v, np.array([[3.0, 8.0]]) / np.sqrt(12.5))
    p = R.probabilities(np.log(np.array([[1.0, 2.0, 5.0]])), np.array([1.0]))
    assert np.allclose(p, [[0.125, 0.25, 0.625]])
    # u q = 0.45 < p = 0.5 keeps token 1; at the end the target's own largest weight / noise
    p = np.array([[[0.5, 0.5], [0.9, 0.1]]])
    q = np.array([[[0.1, 0.9]]])
    tokens, n = R.verify(np.array([[1]]), p, np.array([[0.5]]), np.array([[1.0, 0.01]]), q)
    assert tokens.tolist() == [[1, 1]] and n.tolist() == [1]
    # u q = 0.81 refuses it; only token 0 has weight left over
    tokens, n = R.verify(np.array([[1]]), p, np.array([[0.9]]), np.array([[1.0, 0.01]]), q)
    assert tokens.tolist() == [[0, -1]] and n.tolist() == [0]

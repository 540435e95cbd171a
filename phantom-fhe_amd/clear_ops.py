"""The clear end of an encrypted generation step, on the GPU.

A server that evaluates a model under encryption hands back the ciphertext of a
hidden state; only the holder of the key can turn it into an answer.  These are
the operators the holder runs on decrypted states: the norm, products with clear
weights in 8 bits, probabilities, and the check of drafted tokens (an encrypted
pass takes so long that several drafted tokens are checked per pass).  Callers use
them through pyPhantom, which re-exports them.

They take torch tensors on a GPU, launch on torch's current stream of the tensors'
device, return new tensors (rms_norm_int8 without a residual returns x itself as the
total) and never wait for the GPU.  Rows may be strided, the elements of a row are
adjacent.  Wrong arguments raise ValueError, as everywhere in pyPhantom.  They are for
inference: what they return carries no gradient, whatever its inputs require, and
they take real tensors only, not those of torch's tracing or vmap.  There is no CPU
fallback.
"""
from __future__ import annotations

import torch

import pfa_native as _N

__all__ = ["quantize_int8", "rms_norm_int8", "int8_matmul", "token_probabilities", "verify_drafts"]

_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # PFA_F32, PFA_BF16, PFA_F16
# the handle of the current stream of a device: torch.cuda.current_stream without the object
# around it, which costs a call of a few microseconds more than its launch
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch.cuda.current_device
_WHOLE = {torch.int32: 4, torch.int64: 8}


def _fail(what):
    raise ValueError(what)


def _type_of(t, name):
    code = _TYPE.get(t.dtype)
    if code is None:
        _fail(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    return code


def _same_device(first, *others):
    if not first.is_cuda:
        _fail("expected tensors on a GPU")
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            _fail(f"tensors on {first.device} and on {t.device}")


_entries = {}


def _call(name, t, *args):
    """The entry point on t's device and its current stream."""
    f = _entries.get(name)
    if f is None:
        f = _entries[name] = getattr(_N.lib(), name)
    index = t.get_device()
    if index == _current_device():
        rc = f(*args, _raw_stream(index) or _N.HIP_STREAM_LEGACY)
    else:
        with torch.cuda.device(index):
            rc = f(*args, _raw_stream(index) or _N.HIP_STREAM_LEGACY)
    if rc:
        _N.check(rc)


def _matrix(t, name):
    """(t as a two-dimensional view of its rows, distance between them)."""
    if t.dim() != 2:
        if t.dim() < 1:
            _fail(f"{name} needs at least one dimension")
        t = t.reshape(-1, t.shape[-1]) if t.numel() else t.new_empty((t.shape[:-1].numel(), t.shape[-1]))
    (rows, width), (stride, inner) = t.shape, t.stride()
    if inner != 1 and width > 1:
        _fail(f"{name}: the elements of a row must be adjacent")
    if rows <= 1:
        return t, width
    if 0 < stride < width:
        _fail(f"{name}: rows overlap")
    return t, stride


def _vector(t, n, dtype, name):
    if t.dtype != dtype or t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        _fail(f"{name}: expected {n} adjacent values of {dtype}, got {tuple(t.shape)} of {t.dtype}")
    return t


def _new(like, shape, dtype):
    """An empty contiguous tensor on like's device (the strided call is the cheapest of torch's)."""
    dims = len(shape)
    if dims == 2 and shape[1]:
        strides = (shape[1], 1)
    elif dims == 1:
        strides = (1,)
    else:
        return torch.empty(shape, dtype=dtype, device=like.device)
    return torch.empty_strided(shape, strides, dtype=dtype, device=like.device)


def _new_codes(like):
    """(codes of like's shape, distance of their rows): rows start at whole cache lines, which
    int8_matmul reads fastest (777 x 5003 x 2050 at 2176 bytes a row 18.4 us, at 2064 20.3 us)."""
    shape = like.shape
    width = shape[-1]
    stride = (width + 127) & ~127 if width > 128 else (width + 15) & ~15
    if stride == width or not like.numel():
        return _new(like, shape, torch.int8), width
    strides, step = [1], stride
    for n in shape[-2::-1]:
        strides.append(step)
        step *= n
    # made with these strides at once: a view of whole rows would cost another 1.3 us
    return torch.empty_strided(shape, strides[::-1], dtype=torch.int8, device=like.device), stride


def _workspace(need, device):
    """(tensor to hold on to, address, bytes) of a call's workspace."""
    if not need:
        return None, None, 0
    t = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=device)
    return t, t.data_ptr(), need


def quantize_int8(x):
    """Codes of 8 bits of x [..., width], with one scale for each row: (codes int8
    [..., width], scales float32 [...]), x ~ codes * scales.

    scale = max|x| / 127, rounded to 32 bits, code = 127 x / max|x| to the nearest, ties
    to even.  Rows of zeros have scale 0 (one so small that only its scale rounds to 0
    keeps its codes); rows with a NaN or an infinity have scale NaN and codes 0.  For weights a row is an output channel, for activations a token.  Rows of more
    than 128 codes start at multiples of 128 bytes (codes.stride() says where).
    """
    kind = _type_of(x, "x")
    _same_device(x)
    rows, stride = _matrix(x, "x")
    codes, codes_stride = _new_codes(x)
    n, width = rows.shape
    scales = _new(x, (n,) if x.dim() == 2 else x.shape[:-1], torch.float32)
    if n:
        _call("pfa_quantize_int8", x, rows.data_ptr(), stride, kind, n, width, codes.data_ptr(), codes_stride,
              scales.data_ptr())
    return codes, scales


def rms_norm_int8(x, weight, eps=1e-6, residual=None):
    """Root-mean-square norm of x + residual as codes of 8 bits: (codes int8 [..., width],
    scales float32 [...], total).

    With y = x + residual: total = y in x's type (x itself without a residual), and
    codes, scales are quantize_int8's of y / sqrt(mean(y^2) + eps) * weight, formed from
    the unrounded y.  x [..., width]; residual like x; weight [width]; all of one type.
    y, y weight and the sum of squares are formed in 32 bits: a row where one of them is
    not finite there has scale NaN and codes 0.  The codes are those of y weight (the
    root is common to a row and changes none).
    """
    kind = _type_of(x, "x")
    _same_device(x, weight, residual)
    if not 0 <= eps < float("inf"):
        _fail("eps must be finite and 0 or more")
    rows, stride = _matrix(x, "x")
    n, width = rows.shape
    if width == 0:
        _fail("x: the mean of an empty row")
    _vector(weight, width, x.dtype, "weight")
    total, more, more_stride, total_stride = x, None, 0, 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            _fail(f"residual: expected {tuple(x.shape)} of {x.dtype}, got {tuple(residual.shape)} of {residual.dtype}")
        more, more_stride = _matrix(residual, "residual")
        total, total_stride = _new(x, x.shape, x.dtype), width
    codes, codes_stride = _new_codes(x)
    scales = _new(x, (n,) if x.dim() == 2 else x.shape[:-1], torch.float32)
    if n:
        _call("pfa_rms_norm_int8", x, rows.data_ptr(), stride, more.data_ptr() if more is not None else None,
              more_stride, weight.data_ptr(), kind, n, width, float(eps), total.data_ptr() if total_stride else None,
              total_stride, codes.data_ptr(), codes_stride, scales.data_ptr())
    return codes, scales, total


def int8_matmul(a, a_scales, b, b_scales, bias=None, out_dtype=torch.bfloat16):
    """out[..., n] = (sum_k a[..., k] b[n, k]) a_scales[...] b_scales[n] + bias[n].

    a int8 [..., K] with a_scales float32 [...] (one for each token), b int8 [N, K] with
    b_scales float32 [N] (one for each output channel), as quantize_int8 gives them;
    bias float32 [N]; out of out_dtype (float32, bfloat16 or float16).  The sums are
    exact, so K is at most 131071; scales and bias are applied in 32 bits.  Rows of a
    and b that start at multiples of 128 bytes are read fastest.
    """
    kind = _TYPE.get(out_dtype)
    if kind is None:
        _fail(f"out_dtype: expected float32, bfloat16 or float16, got {out_dtype}")
    if a.dtype != torch.int8 or b.dtype != torch.int8:
        _fail(f"expected int8 codes, got {a.dtype} and {b.dtype}")
    _same_device(a, a_scales, b, b_scales, bias)
    if b.dim() != 2 or a.dim() < 1 or a.shape[-1] != b.shape[1]:
        _fail(f"shapes {tuple(a.shape)} and {tuple(b.shape)} do not multiply")
    if a_scales.dtype != torch.float32 or a_scales.shape != a.shape[:-1] or not a_scales.is_contiguous():
        _fail(f"a_scales: expected contiguous float32 {tuple(a.shape[:-1])}, got {tuple(a_scales.shape)} of "
              f"{a_scales.dtype}")
    rows, a_stride = _matrix(a, "a")
    cols, b_stride = _matrix(b, "b")
    m, k = rows.shape
    n = cols.shape[0]
    _vector(b_scales, n, torch.float32, "b_scales")
    if bias is not None:
        _vector(bias, n, torch.float32, "bias")
    out = _new(a, (*a.shape[:-1], n), out_dtype)
    if m and n:
        held, space, size = _workspace(_N.matmul_workspace(m, n, k), out.device)
        _call("pfa_int8_matmul", a, rows.data_ptr(), a_stride, a_scales.data_ptr(), cols.data_ptr(), b_stride,
              b_scales.data_ptr(), bias.data_ptr() if bias is not None else None, m, n, k, out.data_ptr(), kind, n,
              space, size)
    return out


def token_probabilities(logits, temperature=1.0, mask=None):
    """softmax(logits / temperature) over the allowed places: float32 [..., vocab].

    temperature: a number, or float32 [...] with one for each row; at 0 the lowest place
    of the largest allowed logit gets 1.  mask: bool [vocab] or like logits, True where
    a token is allowed; other places get 0 whatever their logits are.  A row that allows
    nothing (or -infinity alone) is all 0.  A NaN, or above temperature 0 a +infinity, in
    an allowed place and a negative or NaN temperature make a row's allowed places NaN.
    """
    kind = _type_of(logits, "logits")
    rows, stride = _matrix(logits, "logits")
    n, vocab = rows.shape
    temperatures, one = None, 0.0
    if isinstance(temperature, torch.Tensor):
        if temperature.dtype != torch.float32 or temperature.shape != logits.shape[:-1] or \
                not temperature.is_contiguous():
            _fail(f"temperature: expected a number or contiguous float32 {tuple(logits.shape[:-1])}")
        temperatures = temperature
    else:
        one = float(temperature)
        if not 0 <= one < float("inf"):
            _fail("the temperature must be finite and 0 or more")
    allowed, mask_stride = None, 0
    if mask is not None:
        if mask.dtype != torch.bool or (mask.shape != logits.shape and mask.shape != (vocab,)):
            _fail(f"mask: expected bool of {tuple(logits.shape)} or ({vocab},), got {tuple(mask.shape)} of "
                  f"{mask.dtype}")
        if mask.dim() == 1 and vocab > 1 and mask.stride(0) != 1:
            _fail("mask: the places of a row must be adjacent")
        if mask.shape == logits.shape and logits.dim() > 1:
            allowed, mask_stride = _matrix(mask, "mask")
        else:
            allowed = mask
    _same_device(logits, temperatures, mask)
    out = _new(logits, logits.shape, torch.float32)
    if out.numel():
        held, space, size = _workspace(_N.token_workspace(n, vocab), out.device)
        _call("pfa_token_probabilities", logits, rows.data_ptr(), stride, kind, n, vocab,
              temperatures.data_ptr() if temperatures is not None else None, one,
              allowed.data_ptr() if allowed is not None else None, mask_stride, out.data_ptr(), space, size)
    return out


def verify_drafts(draft_tokens, target_probs, uniforms, noise, draft_probs=None, lengths=None):
    """Drafted tokens against the target's probabilities, by given random numbers:
    (tokens [batch, drafts + 1], accepted int32 [batch]).

    draft_tokens int32 or int64 [batch, drafts]; target_probs [batch, drafts + 1, vocab];
    draft_probs [batch, drafts, vocab] of the same type, or None where the drafts were
    certain (chosen without chance); uniforms float32 [batch, drafts] in [0, 1); noise
    float32 [batch, vocab], exponentially distributed; lengths int32 or int64 [batch]: how
    many drafts a sequence has, where not all.

    A draft x is kept while uniform * draft_probs[x] < target_probs[x]; a token outside the
    vocabulary is not.  At the first refusal a token is drawn from max(target - draft, 0),
    at the end of the drafts from target: the one with the largest weight / noise (the
    lowest among equals), whose distribution is the weights'.  So the tokens are distributed
    as if the target had drawn them one by one.  `tokens` are the kept drafts, that
    token, then -1; `accepted` counts the kept drafts.  Where the difference leaves
    nothing, target is taken; where no weight is positive, the token is -1.  With 0 drafts
    this draws one token for each sequence.
    """
    kind = _type_of(target_probs, "target_probs")
    size = _WHOLE.get(draft_tokens.dtype)
    if size is None:
        _fail(f"draft_tokens: expected int32 or int64, got {draft_tokens.dtype}")
    _same_device(target_probs, draft_tokens, uniforms, noise, draft_probs, lengths)
    if target_probs.dim() != 3 or target_probs.shape[1] < 1:
        _fail(f"target_probs: expected [batch, drafts + 1, vocab], got {tuple(target_probs.shape)}")
    batch, places, vocab = target_probs.shape
    drafts = places - 1

    def place(t, name):
        outer, step, inner = t.stride()
        if inner != 1 and vocab > 1:
            _fail(f"{name}: the probabilities of a place must be adjacent")
        return outer, step

    if draft_tokens.shape != (batch, drafts) or not draft_tokens.is_contiguous():
        _fail(f"draft_tokens: expected contiguous {(batch, drafts)}, got {tuple(draft_tokens.shape)}")
    if uniforms.dtype != torch.float32 or uniforms.shape != (batch, drafts) or not uniforms.is_contiguous():
        _fail(f"uniforms: expected contiguous float32 {(batch, drafts)}, got {tuple(uniforms.shape)} of "
              f"{uniforms.dtype}")
    if noise.dtype != torch.float32 or noise.shape != (batch, vocab) or (vocab > 1 and noise.stride(1) != 1):
        _fail(f"noise: expected float32 {(batch, vocab)} with adjacent elements, got {tuple(noise.shape)} of "
              f"{noise.dtype}")
    target_batch, target_place = place(target_probs, "target_probs")
    draft_batch = draft_place = 0
    if draft_probs is not None:
        if draft_probs.shape != (batch, drafts, vocab) or draft_probs.dtype != target_probs.dtype:
            _fail(f"draft_probs: expected {(batch, drafts, vocab)} of {target_probs.dtype}, got "
                  f"{tuple(draft_probs.shape)} of {draft_probs.dtype}")
        draft_batch, draft_place = place(draft_probs, "draft_probs")
    length_size = 4
    if lengths is not None:
        length_size = _WHOLE.get(lengths.dtype)
        if length_size is None or lengths.shape != (batch,) or not lengths.is_contiguous():
            _fail(f"lengths: expected {batch} adjacent values of int32 or int64, got {tuple(lengths.shape)} of "
                  f"{lengths.dtype}")
    tokens = _new(target_probs, (batch, places), draft_tokens.dtype)
    accepted = _new(target_probs, (batch,), torch.int32)
    if batch:
        held, space, need = _workspace(_N.token_workspace(batch, vocab), tokens.device)
        _call("pfa_verify_drafts", target_probs, draft_tokens.data_ptr(), size,
              lengths.data_ptr() if lengths is not None else None, length_size, batch, drafts, vocab,
              target_probs.data_ptr(), target_batch, target_place,
              draft_probs.data_ptr() if draft_probs is not None else None, draft_batch, draft_place, kind,
              uniforms.data_ptr(), noise.data_ptr(), noise.stride(0), tokens.data_ptr(), accepted.data_ptr(), space,
              need)
    return tokens, accepted

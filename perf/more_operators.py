"""More workloads of the clear end of an encrypted generation step: products in 8-bit floating point with a scale for
each block of 128, and log probabilities, through pyPhantom, the framework's public API.

A case is a dict of plain values; its "op" says which operator it is:

  norm      rms_norm_fp8: residual's addition, root-mean-square norm, e4m3 codes with a scale for each 128 of a row
  quant     quantize_fp8: e4m3 codes with a scale for each 1 x 128 (activations) or 128 x 128 (weights)
  matmul    fp8_matmul: product of two matrices of such codes
  logprobs  token_log_probs: log probabilities of given tokens, entropy, the largest alternatives

`own` false computes the same from elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
BLOCK = 128
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_E4M3 = torch.float8_e4m3fn


def _ph():
    ph = sys.modules.get("pyPhantom")
    if ph is None:
        pkg = os.path.join(os.getcwd(), "phantom-fhe_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        import pyPhantom as ph
    return ph


def listed():
    return [
        # the last norm of 4 sequences with 4 drafts and one more place each, in the type that decryption gives
        {"name": "norm_20x4096", "op": "norm", "rows": 20, "width": 4096, "type": "fp32", "residual": True},
        # a long prompt through the norm before a clear layer
        {"name": "norm_4096x8192", "op": "norm", "rows": 4096, "width": 8192, "type": "bf16", "residual": True},
        # a prompt's activations, an odd width whose rows start at any alignment and whose last block is short
        {"name": "quant_777x5119", "op": "quant", "rows": 777, "width": 5119, "type": "fp16", "block": 1},
        # the weights of a layer, laid out when they are loaded
        {"name": "quant_16384x4096", "op": "quant", "rows": 16384, "width": 4096, "type": "bf16", "block": 128},
        # one token through a square layer: the matrix is read once
        {"name": "matmul_1x4096x4096", "op": "matmul", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "bias": False,
         "packed": False},
        # the vocabulary product of 4 sequences with 4 drafts and one more place each
        {"name": "matmul_20x131072x4096", "op": "matmul", "m": 20, "n": 131072, "k": 4096, "type": "fp32",
         "bias": False, "packed": False},
        # 64 sequences of 5 places through a narrowing layer: few tiles, long sums
        {"name": "matmul_320x4096x16384", "op": "matmul", "m": 320, "n": 4096, "k": 16384, "type": "bf16",
         "bias": False, "packed": False},
        # odd everything, with a bias, codes and scales row after row as a file holds them
        {"name": "matmul_777x5003x2050", "op": "matmul", "m": 777, "n": 5003, "k": 2050, "type": "fp16", "bias": True,
         "packed": True},
        # a prompt of 4096 tokens through a widening layer
        {"name": "matmul_4096x16384x4096", "op": "matmul", "m": 4096, "n": 16384, "k": 4096, "type": "bf16",
         "bias": False, "packed": False},
        # one answer with its alternatives
        {"name": "logprobs_1x131072", "op": "logprobs", "rows": 1, "vocab": 131072, "type": "fp32", "mask": "none",
         "given": 1, "top": 20, "heat": False},
        # 64 sequences of 5 places, each with its own allowed tokens and temperature, two answers scored
        {"name": "logprobs_320x32768", "op": "logprobs", "rows": 320, "vocab": 32768, "type": "bf16", "mask": "rows",
         "given": 2, "top": 5, "heat": True},
        # the likelihood of a given text of 2048 tokens
        {"name": "logprobs_2048x131072", "op": "logprobs", "rows": 2048, "vocab": 131072, "type": "bf16",
         "mask": "none", "given": 1, "top": 1, "heat": False},
    ]


def _log(rng, lo, hi):
    """A whole number of lo to hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """Half of them multiples of 128, the others any number."""
    w = _log(rng, lo, hi)
    return max(BLOCK, w // BLOCK * BLOCK) if rng.random() < 0.5 and hi >= BLOCK else w


def draw(rng):
    op = rng.choice(["norm", "quant", "quant", "matmul", "matmul", "matmul", "matmul", "logprobs", "logprobs",
                     "logprobs"])
    if op in ("norm", "quant"):
        width = _width(rng, 64, 16384)
        block = rng.choice([1, 128]) if op == "quant" else 1
        most = (1 << 26) // width if block == 128 else (1 << 25) // width
        c = {"op": op, "rows": _log(rng, 1, min(16384, most)), "width": width,
             "type": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
        if op == "norm":
            c["residual"] = rng.random() < 0.7
        else:
            c["block"] = block
        return c
    if op == "matmul":
        n, k = _width(rng, 64, 131072), _width(rng, 64, 16384)
        while n * k > 1 << 29:
            n //= 2
        return {"op": op, "m": _log(rng, 1, max(1, min(8192, (1 << 37) // (n * k), (1 << 28) // n))), "n": n, "k": k,
                "type": rng.choice(["bf16", "fp16", "fp32"]), "bias": rng.random() < 0.5,
                "packed": rng.random() < 0.3}
    vocab = _width(rng, 1000, 131072)
    return {"op": op, "rows": _log(rng, 1, min(4096, (1 << 27) // vocab)), "vocab": vocab,
            "type": rng.choice(["bf16", "fp16", "fp32"]), "mask": rng.choice(["none", "none", "one", "rows"]),
            "given": rng.choice([1, 1, 2, 5]), "top": rng.choice([0, 1, 5, 20]), "heat": rng.random() < 0.5}


# ------------------------------------------------------------- inputs
def _blocks(n):
    return -(-n // BLOCK)


def _codes(gen, rows, width, packed, dev):
    """Codes of normal values whose blocks' largest are near 448.  Packed: row after row; otherwise rows of more than 128
    start at multiples of 128 bytes, as quantize_fp8 lays them out."""
    step = BLOCK if width > BLOCK else 16
    pitch = width if packed else -(-width // step) * step
    out = torch.zeros((rows, pitch), dtype=torch.uint8, device=dev).view(_E4M3)[:, :width]
    each = max(1, (1 << 26) // max(width, 1))
    for i in range(0, rows, each):
        x = torch.randn((min(each, rows - i), width), device=dev, generator=gen)
        out[i:i + each] = x.mul_(120).clamp_(-448, 448).to(_E4M3)
    return out


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    op, s = case["op"], dict(case)

    def normal(*shape):
        return torch.randn(shape, device=dev, generator=gen)

    def uniform(*shape):
        return torch.rand(shape, device=dev, generator=gen)

    if op in ("norm", "quant"):
        t, rows, width = _TYPES[case["type"]], case["rows"], case["width"]
        # hidden states: rows of different size, some channels far larger than the others
        channel = torch.exp(normal(width) * 0.7)
        s["x"] = (normal(rows, width) * channel * torch.exp(normal(rows, 1) * 0.5)).to(t)
        if op == "norm":
            s["weight"] = (1 + 0.2 * normal(width)).to(t)
            s["r"] = (normal(rows, width) * channel).to(t) if case["residual"] else None
        return s
    if op == "matmul":
        m, n, k, packed = case["m"], case["n"], case["k"], case["packed"]
        s["a"], s["b"] = _codes(gen, m, k, packed, dev), _codes(gen, n, k, packed, dev)
        # activations' scales of a block stand together (quantize_fp8), or those of a row (packed)
        sa = (0.5 + uniform(_blocks(k), m)) / 448
        s["sa"] = sa.t().contiguous() if packed else sa.t()
        s["sb"] = (0.5 + uniform(_blocks(n), _blocks(k))) / (448 * k ** 0.5)
        s["bias"] = normal(n) if case["bias"] else None
        return s
    rows, vocab = case["rows"], case["vocab"]
    s["logits"] = torch.empty((rows, vocab), dtype=_TYPES[case["type"]], device=dev)
    each = max(1, (1 << 27) // vocab)
    for i in range(0, rows, each):
        s["logits"][i:i + each] = normal(min(each, rows - i), vocab).mul_(3)
    s["tokens"] = (uniform(rows, case["given"]) * vocab).long().clamp_(max=vocab - 1)
    if case["given"] == 1:
        s["tokens"] = s["tokens"].squeeze(1)
    s["mask"] = {"none": lambda: None, "one": lambda: uniform(vocab) < 0.5,
                 "rows": lambda: uniform(rows, vocab) < uniform(rows, 1)}[case["mask"]]()
    s["temperature"] = 0.5 + uniform(rows) if case["heat"] else 1.0
    return s


# ------------------------------------------------------------- one pass
def run(s):
    return (_own if own else _plain)(s)


def _spread(scales, width, rows=1):
    """Scales of blocks, one for each column of a row (and for each row, in blocks of more than one)."""
    out = scales.repeat_interleave(BLOCK, 1)[:, :width]
    return out if rows == 1 else out.repeat_interleave(BLOCK, 0)


def _values(codes, scales, like, block):
    """What codes of 8 bits stand for, in the input's type."""
    (rows, width), out = codes.shape, codes.to(like if like != torch.float16 else torch.float32)
    if width % BLOCK == 0 and rows % block == 0:
        whole = out.view(rows // block, block, width // BLOCK, BLOCK)
        whole.mul_(scales[:, None, :, None])
    else:
        out.mul_(_spread(scales, width, block)[:rows])
    return out.to(like)


def _own(s):
    ph, op = _ph(), s["op"]
    if op == "norm":
        codes, scales, total = ph.rms_norm_fp8(s["x"], s["weight"], EPS, s["r"])
        return [_values(codes, scales, s["x"].dtype, 1), scales] + ([total] if s["r"] is not None else [])
    if op == "quant":
        codes, scales = ph.quantize_fp8(s["x"], s["block"])
        return [_values(codes, scales, s["x"].dtype, s["block"]), scales]
    if op == "matmul":
        return [ph.fp8_matmul(s["a"], s["sa"], s["b"], s["sb"], s["bias"], _TYPES[s["type"]])]
    return list(ph.token_log_probs(s["logits"], s["tokens"], s["top"], s["temperature"], s["mask"]))


def _plain_codes(x, block):
    """(codes, scales) of x in 32 bits: the scale is the least power of two that takes a block's largest to 448 or less."""
    rows, width = x.shape
    down, across = -(-rows // block), _blocks(width)
    whole = torch.nn.functional.pad(x, (0, across * BLOCK - width, 0, down * block - rows))
    whole = whole.view(down, block, across, BLOCK)
    top = whole.abs().amax((1, 3))
    part, power = torch.frexp(top)  # part of 0.5 to 1: 448 is 0.875 2^9
    power = torch.where(part > 0.875, power - 8, power - 9).clamp(min=-126)
    scales = torch.where(top > 0, torch.ldexp(torch.ones_like(top), power), 0.0)
    codes = whole / torch.where(scales > 0, scales, 1.0)[:, None, :, None]
    return codes.view(down * block, across * BLOCK)[:rows, :width].to(_E4M3), scales


def _plain(s):
    op = s["op"]
    if op == "quant":
        codes, scales = _plain_codes(s["x"].float(), s["block"])
        return [_values(codes, scales, s["x"].dtype, s["block"]), scales]
    if op == "norm":
        y, t, total = s["x"].float(), s["x"].dtype, []
        if s["r"] is not None:
            y = y + s["r"].float()
            total = [y.to(t)]
        codes, scales = _plain_codes(y * s["weight"].float(), 1)
        scales = scales * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
        return [_values(codes, scales, t, 1), scales] + total
    if op == "matmul":
        (m, k), n = s["a"].shape, s["b"].shape[0]
        a = s["a"].float() * _spread(s["sa"], k)
        b = s["b"].float() * _spread(s["sb"], k, BLOCK)[:n]
        y = a @ b.t()
        if s["bias"] is not None:
            y = y + s["bias"]
        return [y.to(_TYPES[s["type"]])]
    x, tokens = s["logits"].float(), s["tokens"]
    if s["mask"] is not None:
        x = torch.where(s["mask"], x, -torch.inf)
    heat = s["temperature"].unsqueeze(-1) if isinstance(s["temperature"], torch.Tensor) else s["temperature"]
    largest = x.amax(-1, keepdim=True)
    base = torch.where(largest == -torch.inf, 0.0, largest)
    d = (x - base) / heat
    w = torch.exp(d)
    total = w.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total - torch.where(w > 0, w * d, 0.0).sum(-1, keepdim=True) / total
    entropy = torch.where(total > 0, entropy, 0.0).squeeze(-1)
    del w

    def log_probs(at):
        return torch.where(total > 0, torch.gather(d, 1, at) - log_total, -torch.inf)

    given = log_probs(tokens.view(x.shape[0], -1)).view(tokens.shape)
    tops, places = [x.new_empty((x.shape[0], 0))], [tokens.new_empty((x.shape[0], 0))]
    for _ in range(s["top"]):  # the lowest place among equals, then without it
        at = x.argmax(-1, keepdim=True)
        there = torch.gather(x, 1, at) > -torch.inf
        tops.append(torch.where(there, log_probs(at), -torch.inf))
        places.append(torch.where(there, at, -1))
        x = x.scatter(1, at, -torch.inf)
    return [given, entropy, torch.cat(tops, 1), torch.cat(places, 1)]


# ------------------------------------------------------------- what a pass cannot do without
def work(case):
    """Bytes: every operand once, the results once (codes in 8 bits, a scale a block).  Operations: one for each product,
    sum, comparison or exponential."""
    op = case["op"]
    if op in ("norm", "quant"):
        size, n = _TYPES[case["type"]].itemsize, case["rows"] * case["width"]
        moved = size * (3 if case.get("residual") else 1) + 1
        block = case.get("block", 1)
        scales = 4 * -(-case["rows"] // block) * _blocks(case["width"])
        return {"bytes": n * moved + scales + (size * case["width"] if op == "norm" else 0),
                "flops": n * (8 if op == "norm" else 3)}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        scales = 4 * (m + _blocks(n)) * _blocks(k)
        return {"bytes": (m + n) * k + scales + m * n * _TYPES[case["type"]].itemsize + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    n = case["rows"] * case["vocab"]
    masks = {"none": 0, "one": case["vocab"], "rows": n}[case["mask"]]
    each = 12 * case["given"] + 12 * case["top"] + 4 + (4 if case["heat"] else 0)
    return {"bytes": n * _TYPES[case["type"]].itemsize + masks + each * case["rows"], "flops": 6 * n}


def exact(case, seed):
    """The floating outputs from the definitions, in 64 bits."""
    s, op = prepare(case, seed), case["op"]
    if op == "matmul":
        (m, k), n = s["a"].shape, s["b"].shape[0]
        at = torch.arange(k, device=s["a"].device) // BLOCK
        a = s["a"].float().double() * s["sa"].double()[:, at]
        y = torch.empty((m, n), dtype=torch.float64, device=a.device)
        for i in range(0, n, 8192):
            b = s["b"][i:i + 8192].float().double()
            rows = torch.arange(i, i + b.shape[0], device=a.device) // BLOCK
            y[:, i:i + 8192] = torch.mm(a, b.mul_(s["sb"].double()[rows][:, at]).t().contiguous())
        return [y if s["bias"] is None else y.add_(s["bias"].double()[None, :])]
    if op in ("norm", "quant"):
        h, total, factor = s["x"].double(), [], 1.0
        if op == "norm":
            if s["r"] is not None:
                h = h + s["r"].double()
                total = [h]
            factor = 1 / torch.sqrt(h.pow(2).sum(1, keepdim=True) / case["width"] + EPS)
            h = h * s["weight"].double()
        rows, width = h.shape
        block = case.get("block", 1)
        values = torch.empty_like(h)
        steps = torch.zeros((-(-rows // block), _blocks(width)), dtype=torch.float64, device=h.device)
        for j in range(_blocks(width)):
            part = h[:, j * BLOCK:(j + 1) * BLOCK]
            tops = part.abs().max(1).values
            if block > 1:
                tops = torch.nn.functional.pad(tops, (0, steps.shape[0] * block - rows)).view(-1, block).max(1).values
            step = torch.exp2(torch.ceil(torch.log2(tops / 448)).clamp(min=-126))
            # logarithms are rounded: the least power that holds the largest
            step = torch.where(step / 2 * 448 >= tops, step / 2, step)
            step = torch.where(step * 448 < tops, step * 2, step).clamp(min=2.0 ** -126)
            steps[:, j] = torch.where(tops > 0, step, torch.zeros_like(step))
            q = part / step.repeat_interleave(block)[:rows, None]
            # e4m3: 4 significant bits, from 2^-6 downwards steps of 2^-9
            ulp = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
            values[:, j * BLOCK:(j + 1) * BLOCK] = torch.round(q / ulp) * ulp * step.repeat_interleave(block)[:rows, None]
        return [values * factor, steps * factor] + total
    outs = []
    each = max(1, (1 << 26) // case["vocab"])
    for i in range(0, case["rows"], each):
        z = s["logits"][i:i + each].double()
        mask = s["mask"]
        if mask is not None:
            z = z.masked_fill(~(mask if mask.dim() == 1 else mask[i:i + each]), float("-inf"))
        if case["heat"]:
            z = z / s["temperature"][i:i + each].double()[:, None]
        z = torch.nan_to_num_(z - torch.logsumexp(z, 1, keepdim=True), nan=float("-inf"), neginf=float("-inf"))
        p = torch.exp(z)
        tokens = s["tokens"][i:i + each]
        given = torch.take_along_dim(z, tokens.reshape(tokens.shape[0], -1), 1).reshape(tokens.shape)
        outs.append([given, -(p * z.clamp_min(-1e4)).sum(1), torch.topk(z, case["top"], 1).values])
    return [torch.cat(v) for v in zip(*outs)] + [None]

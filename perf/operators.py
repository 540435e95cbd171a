"""The workloads of the clear end of an encrypted generation step: what the holder of the key runs on decrypted hidden
states, through pyPhantom, the framework's public API.

A case is a dict of plain values; its "op" says which operator it is:

  norm      rms_norm_int8: residual's addition, root-mean-square norm, codes of 8 bits with a scale for each row
  quant     quantize_int8: codes of 8 bits with a scale for each row
  matmul    int8_matmul: product of two matrices of such codes
  probs     token_probabilities: logits to probabilities, with a temperature and allowed places
  verify    verify_drafts: drafted tokens against the target's probabilities

`own` false computes the same from elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


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
        # the last norm of a single decoded token: nothing but latency
        {"name": "norm_1x4096", "op": "norm", "rows": 1, "width": 4096, "type": "bf16", "residual": True},
        # a whole prompt through the norm before a clear layer
        {"name": "norm_4096x8192", "op": "norm", "rows": 4096, "width": 8192, "type": "bf16", "residual": True},
        # activations of a few drafted tokens, an odd width whose rows start at any alignment
        {"name": "quant_20x5119", "op": "quant", "rows": 20, "width": 5119, "type": "fp16"},
        # a prompt's activations before the product that narrows them again
        {"name": "quant_2048x16384", "op": "quant", "rows": 2048, "width": 16384, "type": "bf16"},
        # one token through a square layer: the matrix is read once
        {"name": "matmul_1x4096x4096", "op": "matmul", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "bias": False,
         "packed": True},
        # the vocabulary product of 4 sequences with 4 drafts and one more place each
        {"name": "matmul_20x131072x4096", "op": "matmul", "m": 20, "n": 131072, "k": 4096, "type": "fp32",
         "bias": False, "packed": True},
        # odd everything, with a bias, rows padded to 16 bytes as quantize_int8 lays them out
        {"name": "matmul_777x5003x2050", "op": "matmul", "m": 777, "n": 5003, "k": 2050, "type": "fp16", "bias": True,
         "packed": False},
        # a prompt of 4096 tokens through a widening layer
        {"name": "matmul_4096x16384x4096", "op": "matmul", "m": 4096, "n": 16384, "k": 4096, "type": "bf16",
         "bias": False, "packed": True},
        # one sequence: 4 drafts and one more place
        {"name": "probs_5x131072", "op": "probs", "rows": 5, "vocab": 131072, "type": "fp32", "mask": "none"},
        # 64 sequences of 5 places, each with its own allowed tokens
        {"name": "probs_320x32768", "op": "probs", "rows": 320, "vocab": 32768, "type": "bf16", "mask": "rows"},
        # one sequence, 4 drafts
        {"name": "verify_1x4x131072", "op": "verify", "batch": 1, "drafts": 4, "vocab": 131072, "ragged": False,
         "certain": False},
        # 64 sequences with up to 7 drafts each
        {"name": "verify_64x7x100003", "op": "verify", "batch": 64, "drafts": 7, "vocab": 100003, "ragged": True,
         "certain": False},
    ]


def _log(rng, lo, hi):
    """A whole number of lo to hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """Half of them multiples of 128, the others any number."""
    w = _log(rng, lo, hi)
    w = max(128, w // 128 * 128) if rng.random() < 0.5 and hi >= 128 else w
    return w if w != 3072 else w + 128


def draw(rng):
    op = rng.choice(["norm", "norm", "quant", "matmul", "matmul", "matmul", "probs", "probs", "verify", "verify"])
    kind = rng.choice(["bf16", "bf16", "fp16"])
    if op in ("norm", "quant"):
        width = _width(rng, 64, 16384)
        c = {"op": op, "rows": _log(rng, 1, min(8192, (1 << 25) // width)), "width": width, "type": kind}
        if op == "norm":
            c["residual"] = rng.random() < 0.7
        return c
    if op == "matmul":
        n, k = _width(rng, 64, 131072), _width(rng, 64, 16384)
        while n * k > 1 << 29:
            n //= 2
        return {"op": op, "m": _log(rng, 1, max(1, min(8192, (1 << 37) // (n * k), (1 << 28) // n))), "n": n, "k": k,
                "type": rng.choice(["bf16", "fp16", "fp32"]), "bias": rng.random() < 0.5,
                "packed": rng.random() < 0.5}
    vocab = _width(rng, 1000, 131072)
    if op == "probs":
        return {"op": op, "rows": _log(rng, 1, min(512, (1 << 25) // vocab)), "vocab": vocab,
                "type": rng.choice(["bf16", "fp16", "fp32"]), "mask": rng.choice(["none", "one", "rows"])}
    drafts = rng.randint(0, 8)
    return {"op": op, "batch": _log(rng, 1, min(128, (1 << 27) // (vocab * (2 * drafts + 2)))), "drafts": drafts,
            "vocab": vocab, "ragged": rng.random() < 0.5, "certain": rng.random() < 0.3}


# ------------------------------------------------------------- inputs
def _rows16(codes):
    """The same codes with rows that start at multiples of 16 bytes."""
    m, k = codes.shape
    buf = torch.zeros((m, -(-k // 16) * 16), dtype=torch.int8, device=codes.device)
    buf[:, :k] = codes
    return buf[:, :k]


def _codes(gen, rows, width, dev):
    """Codes of rows of normal values whose largest is near 127."""
    out = torch.empty((rows, width), dtype=torch.int8, device=dev)
    step = max(1, (1 << 26) // max(width, 1))
    for i in range(0, rows, step):
        x = torch.randn((min(step, rows - i), width), device=dev, generator=gen)
        out[i:i + step] = x.mul_(32).round_().clamp_(-127, 127).to(torch.int8)
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
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["b"] = _codes(gen, m, k, dev), _codes(gen, n, k, dev)
        if not case["packed"]:
            s["a"], s["b"] = _rows16(s["a"]), _rows16(s["b"])
        s["sa"], s["sb"] = (0.5 + uniform(m)) / 127, (0.5 + uniform(n)) / (127 * k ** 0.5)
        s["bias"] = normal(n) if case["bias"] else None
        return s
    if op == "probs":
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = (normal(rows, vocab) * 3).to(_TYPES[case["type"]])
        s["mask"] = {"none": lambda: None, "one": lambda: uniform(vocab) < 0.5,
                     "rows": lambda: uniform(rows, vocab) < uniform(rows, 1)}[case["mask"]]()
        s["temperature"] = 0.5 + uniform(rows)
        return s
    batch, drafts, vocab = case["batch"], case["drafts"], case["vocab"]
    logits = normal(batch, drafts + 1, vocab) * 3
    s["p"] = torch.softmax(logits, -1)
    # a small model's view of the same places
    q = torch.softmax(logits[:, :drafts] + 0.4 * normal(batch, drafts, vocab), -1)
    pick = q if not case["certain"] else s["p"][:, :drafts]
    race = -torch.log1p(-uniform(batch, drafts, vocab))
    s["x"] = (pick / race).argmax(-1) if drafts else torch.zeros((batch, 0), dtype=torch.int64, device=dev)
    s["q"] = None if case["certain"] else q
    s["u"] = uniform(batch, drafts)
    s["e"] = -torch.log1p(-uniform(batch, vocab)) + 1e-10
    s["lengths"] = (uniform(batch) * (drafts + 1)).to(torch.int32).clamp_(max=drafts) if case["ragged"] else None
    return s


# ------------------------------------------------------------- one pass
def run(s):
    return (_own if own else _plain)(s)


def _values(codes, scales, like):
    """What codes of 8 bits stand for, in the input's type."""
    return torch.mul(codes, scales.unsqueeze(-1), out=torch.empty(codes.shape, dtype=like, device=codes.device))


def _own(s):
    ph, op = _ph(), s["op"]
    if op == "norm":
        codes, scales, total = ph.rms_norm_int8(s["x"], s["weight"], EPS, s["r"])
        return [_values(codes, scales, s["x"].dtype), scales] + ([total] if s["r"] is not None else [])
    if op == "quant":
        codes, scales = ph.quantize_int8(s["x"])
        return [_values(codes, scales, s["x"].dtype), scales]
    if op == "matmul":
        return [ph.int8_matmul(s["a"], s["sa"], s["b"], s["sb"], s["bias"], _TYPES[s["type"]])]
    if op == "probs":
        return [ph.token_probabilities(s["logits"], s["temperature"], s["mask"])]
    return list(ph.verify_drafts(s["x"], s["p"], s["u"], s["e"], s["q"], s["lengths"]))


def _plain(s):
    op = s["op"]
    if op in ("norm", "quant"):
        x, t, total = s["x"].float(), s["x"].dtype, []
        if op == "norm":
            if s["r"] is not None:
                x = x + s["r"].float()
                total = [x.to(t)]
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"].float()
        scales = x.abs().amax(-1) / 127
        scale = scales.unsqueeze(-1)
        codes = torch.where(scale > 0, torch.round(x / scale), 0.0)
        return [(codes * scale).to(t), scales] + total
    if op == "matmul":
        y = (s["a"].float() @ s["b"].float().t()) * s["sa"].unsqueeze(-1) * s["sb"]
        if s["bias"] is not None:
            y = y + s["bias"]
        return [y.to(_TYPES[s["type"]])]
    if op == "probs":
        x = s["logits"].float() / s["temperature"].unsqueeze(-1)
        if s["mask"] is not None:
            x = torch.where(s["mask"], x, -torch.inf)
        top = x.amax(-1, keepdim=True)
        x = torch.exp(x - torch.where(top == -torch.inf, 0.0, top))
        total = x.sum(-1, keepdim=True)
        return [torch.where(total > 0, x / total, 0.0)]
    p, q, x, u = s["p"], s["q"], s["x"], s["u"]
    batch, drafts = x.shape
    row = torch.arange(batch, device=p.device)
    place = torch.arange(drafts, device=p.device)
    px = torch.gather(p[:, :drafts], 2, x.unsqueeze(-1)).squeeze(-1)
    qx = torch.gather(q, 2, x.unsqueeze(-1)).squeeze(-1) if q is not None else torch.ones_like(px)
    ends = torch.full((batch,), drafts, device=p.device) if s["lengths"] is None else s["lengths"]
    fine = (u * qx < px) & (place < ends.unsqueeze(-1))
    n = torch.cumprod(fine, 1).sum(1)
    pn = p[row, n]
    if drafts:
        last = n.clamp(max=drafts - 1)
        if q is not None:
            less = pn - q[row, last]
        else:
            less = torch.where(torch.arange(p.shape[2], device=p.device) == x[row, last].unsqueeze(-1), 0.0, pn)
        w = torch.where((n < ends).unsqueeze(-1), less, pn)
        w = torch.where((w > 0).any(-1, keepdim=True), w, pn)
    else:
        w = pn
    best, token = torch.where(w > 0, w / s["e"], 0.0).max(-1)
    token = torch.where(best > 0, token, -1)
    place = torch.arange(drafts + 1, device=p.device)
    padded = torch.nn.functional.pad(x, (0, 1), value=-1)
    at = n.unsqueeze(-1)
    tokens = torch.where(place < at, padded, torch.where(place == at, token.unsqueeze(-1), -1))
    return [tokens, n.to(torch.int32)]


# ------------------------------------------------------------- what a pass cannot do without
def work(case):
    """Bytes: every operand once, the results once (codes in 8 bits; of the probabilities to verify, the row that the
    last token is chosen from).  Operations: one for each product, sum, comparison or exponential."""
    op = case["op"]
    if op in ("norm", "quant"):
        size, n = _TYPES[case["type"]].itemsize, case["rows"] * case["width"]
        moved = size * (3 if case.get("residual") else 1) + 1
        return {"bytes": n * moved + 4 * case["rows"] + (size * case["width"] if op == "norm" else 0),
                "flops": n * (8 if op == "norm" else 3)}
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * (k + 4) + m * n * _TYPES[case["type"]].itemsize + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if op == "probs":
        n = case["rows"] * case["vocab"]
        masks = {"none": 0, "one": case["vocab"], "rows": n}[case["mask"]]
        return {"bytes": n * (_TYPES[case["type"]].itemsize + 4) + masks + 4 * case["rows"], "flops": 5 * n}
    n = case["batch"] * case["vocab"]
    rows = 2 if case["certain"] or not case["drafts"] else 3
    return {"bytes": 4 * n * rows + case["batch"] * case["drafts"] * 20, "flops": 4 * n}


def exact(case, seed):
    """The floating outputs from the definitions, in 64 bits."""
    s, op = prepare(case, seed), case["op"]
    if op == "verify":
        return None  # whole numbers
    if op == "matmul":
        if 2.0 * case["m"] * case["n"] * case["k"] > 3e13:
            return None
        y = torch.empty((case["m"], case["n"]), dtype=torch.float64, device=s["a"].device)
        a = s["a"].double()
        for i in range(0, case["n"], 8192):
            y[:, i:i + 8192] = torch.mm(a, s["b"][i:i + 8192].double().t().contiguous())
        y.mul_(s["sa"].double()[:, None]).mul_(s["sb"].double()[None, :])
        return [y if s["bias"] is None else y.add_(s["bias"].double()[None, :])]
    if op == "probs":
        z = s["logits"].double() / s["temperature"].double()[:, None]
        if s["mask"] is not None:
            z = z.masked_fill(~s["mask"], float("-inf"))
        z = torch.exp(z - torch.logsumexp(z, 1, keepdim=True))
        return [z.nan_to_num_(nan=0.0)]
    h, total = s["x"].double(), None
    if op == "norm":
        if s["r"] is not None:
            h = total = h + s["r"].double()
        h = s["weight"].double() * (h / torch.sqrt(h.pow(2).sum(1, keepdim=True) / case["width"] + EPS))
    step = h.abs().max(1).values / 127
    values = torch.round(h / step.clamp_min(1e-300)[:, None]) * step[:, None]
    return [values, step] + ([total] if total is not None else [])

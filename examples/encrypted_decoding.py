"""Generation with an encrypted layer, both ends of it: python examples/encrypted_decoding.py

The holder of the key drafts tokens with a small clear model, encrypts the hidden states of
all drafted places, and the server applies its matrix to the ciphertexts (a BSGS matrix-vector
product each).  The holder decrypts, adds the residual, and finishes the step in the clear:
norm, vocabulary product in 8 bits, probabilities, and the check of the drafts, which keeps
several tokens for one round trip.  All weights are random; the program compares its
probabilities with the same step in double precision and prints what was kept.
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "phantom-fhe_amd"))
import pyPhantom as ph  # noqa: E402

EPS, TEMPERATURE = 1e-6, 0.8


class Server:
    """Holds a matrix and evaluation keys, sees ciphertexts only."""

    def __init__(self, ctx, enc, glk, matrix, baby, scale):
        n = matrix.shape[0]
        self.ctx, self.glk = ctx, glk
        self.diagonals = ph.pre_encode_bsgs_diagonals(ctx, enc, matrix, n, n, n, baby, scale)

    def layer(self, ct):
        return ph.bsgs_matmul_preencoded(self.ctx, self.glk, ct, self.diagonals)


class Holder:
    """Holds the secret key, the embedding, the last norm's gain and the vocabulary matrix."""

    def __init__(self, ctx, enc, sk, embedding, gain, vocabulary, scale):
        self.ctx, self.enc, self.sk, self.scale = ctx, enc, sk, scale
        self.embedding, self.gain = embedding, gain
        self.codes, self.scales = ph.quantize_int8(vocabulary)  # laid out once

    def encrypt(self, states):
        slots = self.enc.slot_count()
        return [self.sk.encrypt_symmetric(self.ctx, self.enc.encode_double_vector(
            self.ctx, np.tile(v, slots // v.size), self.scale)) for v in states.double().cpu().numpy()]

    def decrypt(self, cts, width):
        rows = [np.array(self.enc.decode_double_vector(self.ctx, self.sk.decrypt(self.ctx, ct)))[:width] for ct in cts]
        return torch.from_numpy(np.stack(rows)).float().to(self.embedding.device)

    def finish(self, states, residual, drafts, draft_probs, uniforms, noise):
        """Decrypted states [places, width] to (tokens, how many drafts were kept, probabilities)."""
        codes, scales, _ = ph.rms_norm_int8(states, self.gain, EPS, residual)
        logits = ph.int8_matmul(codes, scales, self.codes, self.scales, None, torch.float32)
        probs = ph.token_probabilities(logits, TEMPERATURE)
        tokens, kept = ph.verify_drafts(drafts[None], probs[None], uniforms[None], noise[None], draft_probs[None])
        return tokens[0], kept[0], probs


def draft(embedding, head, last, places, gen):
    """`places` tokens one after the other from a small clear model: (tokens, its probabilities)."""
    tokens, probs = [], []
    for _ in range(places):
        state = embedding[last]
        p = ph.token_probabilities((state @ head)[None], TEMPERATURE)
        noise = torch.empty(p.shape, device=p.device).exponential_(generator=gen)
        none = torch.empty((1, 0), device=p.device)
        pick, _ = ph.verify_drafts(none.long(), p[None], none, noise)  # no drafts: one token from p
        last = pick[0, 0]
        tokens.append(last)
        probs.append(p[0])
    return torch.stack(tokens), torch.stack(probs)


def run(logn=13, width=256, vocab=1000, places=4, rounds=6, seed=1, say=print):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    rng = np.random.default_rng(seed)
    ph.set_seed(seed)
    scale, n, baby = 2.0 ** 40, 1 << logn, 16
    p = ph.params(ph.scheme_type.ckks)
    p.set_poly_modulus_degree(n)
    p.set_coeff_modulus(ph.create_coeff_modulus(n, [60, 40, 60]))
    p.set_special_modulus_size(1)
    p.set_galois_elts(ph.get_elts_from_steps(ph.bsgs_required_steps(baby), n))
    ctx = ph.context(p)
    enc, sk = ph.ckks_encoder(ctx), ph.secret_key(ctx)

    matrix = rng.standard_normal((width, width)) / width ** 0.5
    embedding = torch.randn((vocab, width), device=dev, generator=gen)
    gain = 1 + 0.1 * torch.randn(width, device=dev, generator=gen)
    vocabulary = torch.randn((vocab, width), device=dev, generator=gen) / width ** 0.5
    # the small model knows the layer and the vocabulary matrix roughly
    rough = (torch.eye(width, device=dev) + torch.from_numpy(matrix).float().to(dev)).t() @ vocabulary.t()
    head = rough / 2 ** 0.5 + 0.3 * torch.randn((width, vocab), device=dev, generator=gen) / width ** 0.5

    server = Server(ctx, enc, sk.create_galois_keys(ctx), matrix, baby, scale)
    holder = Holder(ctx, enc, sk, embedding, gain, vocabulary, scale)
    last, text, worst = torch.tensor(0, device=dev), [], 0.0
    for _ in range(rounds):
        drafts, draft_probs = draft(embedding, head, last, places, gen)
        states = embedding[torch.cat([last[None], drafts])]  # the last token and every draft
        answers = holder.decrypt([server.layer(ct) for ct in holder.encrypt(states)], width)
        uniforms = torch.rand(places, device=dev, generator=gen)
        noise = torch.empty(vocab, device=dev).exponential_(generator=gen)
        tokens, kept, probs = holder.finish(answers, states, drafts, draft_probs, uniforms, noise)

        # the same step in double precision, nothing encrypted and nothing in 8 bits
        y = states.double() + states.double() @ torch.from_numpy(matrix).to(dev).t()
        y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * gain.double()
        want = torch.softmax(y @ vocabulary.double().t() / TEMPERATURE, -1)
        worst = max(worst, float((probs.double() - want).abs().sum(-1).max()) / 2)
        new = [int(t) for t in tokens if t >= 0]
        text += new
        last = tokens[kept.long()]
        say(f"drafted {drafts.tolist()}, kept {int(kept)}, new tokens {new}")
    say(f"{len(text)} tokens in {rounds} encrypted rounds; probabilities within {worst:.4f} (total variation) of double "
        "precision")
    return text, worst


if __name__ == "__main__":
    run()

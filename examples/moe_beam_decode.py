"""Beam search through a small mixture-of-experts decoder with 4-bit weights:
router -> experts, 4-bit projections and head -> selection over beams and
vocabulary -> the caches and histories follow their parents.

    python examples/moe_beam_decode.py [--batch 4] [--beams 4] [--steps 32]

The weights are random, so the text means nothing; the tokens stay ids.  At the
end each request's best hypothesis is fed through the decoder again, alone and
without any reordering, and its score compared.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from hi_amd._lib import check, load  # noqa: E402
from hi_amd.beam import BeamSearch, reorder_states  # noqa: E402
from hi_amd.moe import MoeExperts  # noqa: E402
from hi_amd.w4 import W4Linear, quantize_w4  # noqa: E402


class Decoder:
    """``layers`` blocks of attention and experts over ``rows`` sequences, one
    token of each at a time, on a stream of the caller's (the router's call
    takes no default stream).  The cache is one tensor [2 * layers][rows]
    [heads][max_len][head_dim], so one call reorders all of it."""

    def __init__(self, rows, max_len, vocab=32000, hidden=1024, heads=8, layers=2, experts=32, top_k=4, inter=512,
                 group=64, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, scale=1.0):
            return torch.randn(*shape, generator=g, device="cuda") * scale

        def w4(n, k):
            return W4Linear(*quantize_w4(normal(n, k, scale=k ** -0.5), group, symmetric=False))

        self.rows, self.max_len, self.vocab, self.hidden, self.heads = rows, max_len, vocab, hidden, heads
        self.layers, self.experts, self.top_k, self.dim = layers, experts, top_k, hidden // heads
        self.embed = normal(vocab, hidden).bfloat16()
        self.places = normal(max_len, hidden, scale=0.2).bfloat16()
        self.qkv = [w4(3 * hidden, hidden) for _ in range(layers)]
        self.proj = [w4(hidden, hidden) for _ in range(layers)]
        self.router = [normal(experts, hidden, scale=hidden ** -0.5) for _ in range(layers)]
        self.moe = [MoeExperts(normal(experts, 2 * inter, hidden, scale=hidden ** -0.5).bfloat16(),
                               normal(experts, hidden, inter, scale=inter ** -0.5).bfloat16(), rows, top_k)
                    for _ in range(layers)]
        self.head = w4(vocab, hidden)
        self.cache = torch.zeros(2 * layers, rows, heads, max_len, self.dim, dtype=torch.bfloat16, device="cuda")
        self.ids = torch.empty(rows, top_k, dtype=torch.int32, device="cuda")
        self.weights = torch.empty(rows, top_k, dtype=torch.float32, device="cuda")
        self.logits = torch.empty(rows, vocab, dtype=torch.float32, device="cuda")

    @staticmethod
    def norm(x):
        x = x.float()
        return x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-6)

    def attend(self, layer, x, at):
        rows, heads, dim = self.rows, self.heads, self.dim
        q, k, v = self.qkv[layer](x.bfloat16()).view(rows, 3, heads, dim).unbind(1)
        keys, values = self.cache[2 * layer], self.cache[2 * layer + 1]
        keys[:, :, at], values[:, :, at] = k.bfloat16(), v.bfloat16()
        score = (keys[:, :, :at + 1].float() * q[:, :, None]).sum(3) * dim ** -0.5
        p = torch.softmax(score, 2)
        return (values[:, :, :at + 1].float() * p[..., None]).sum(2).reshape(rows, heads * dim)

    def route(self, layer, x):
        scores = (x[:, None] * self.router[layer]).sum(2)
        check(load().hi_rocm_launch_moe_topk_router(
            scores.data_ptr(), self.ids.data_ptr(), self.weights.data_ptr(), 0, self.rows, self.experts, self.top_k, 1,
            0, 1.0, torch.cuda.current_stream().cuda_stream))
        return self.ids, self.weights

    def step(self, tokens, at):
        """Logits [rows][vocab] after ``tokens`` (int32 [rows]) at position ``at``."""
        x = (self.embed[tokens.long()] + self.places[at]).float()
        for layer in range(self.layers):
            x = x + self.proj[layer](self.attend(layer, self.norm(x), at).bfloat16())
            y = self.norm(x)
            x = x + self.moe[layer](y.bfloat16(), *self.route(layer, y))
        return self.head(self.norm(x).bfloat16(), out=self.logits)


def beam_decode(model, prompts, beams, steps, eos):
    """The hypotheses of each request in order: (histories int32 [batch][beams]
    [prompt + steps], scores [batch][beams], finished).  ``prompts`` int32
    [batch][length]."""
    batch, start = prompts.shape
    search = BeamSearch(batch, beams, model.vocab)
    rows = batch * beams
    hist = torch.full((rows, start + steps), eos, dtype=torch.int32, device="cuda")
    hist[:, :start] = prompts.repeat_interleave(beams, 0)
    for at in range(start - 1):
        model.step(hist[:, at], at)
    # all beams of a request begin equal: only the first may be extended
    scores = torch.full((batch, beams), -torch.inf, device="cuda")
    scores[:, 0] = 0.0
    finished = torch.zeros(batch, beams, dtype=torch.uint8, device="cuda")
    turns = [search.outputs(batch), search.outputs(batch)]
    lengths = torch.empty(batch, dtype=torch.int32, device="cuda")
    for i in range(steps):
        at = start - 1 + i
        logits = model.step(hist[:, at], at)
        out = search.select(logits, scores, finished=finished, eos_id=eos, out=turns[i % 2])
        parents = out["parents"]
        if i + 1 < steps:  # (no step reads the cache any more)
            lengths.fill_(at + 1)
            reorder_states(model.cache, parents, row_dim=1, length_dim=3, lengths=lengths)
        reorder_states(hist, parents)
        hist[:, at + 1] = out["tokens"].view(-1)
        scores, finished = out["scores"], out["finished"]
    return hist.view(batch, beams, -1), scores, finished


def rescore(model, hypotheses, start, eos):
    """Scores of whole sequences (int32 [rows][length]) fed one token after
    another, in double precision from the decoder's logits."""
    score = torch.zeros(hypotheses.shape[0], dtype=torch.float64, device="cuda")
    done = torch.zeros_like(score, dtype=torch.bool)
    for at in range(hypotheses.shape[1] - 1):
        logits = model.step(hypotheses[:, at], at)
        if at + 1 < start:
            continue
        token = hypotheses[:, at + 1].long()
        step = torch.log_softmax(logits.double(), 1).gather(1, token[:, None])[:, 0]
        score = torch.where(done, score, score + step)
        done |= token == eos
    return score


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--batch", type=int, default=4)
    p.add_argument("--beams", type=int, default=4)
    p.add_argument("--steps", type=int, default=32)
    a = p.parse_args()
    prompt, eos = 4, 2
    model = Decoder(a.batch * a.beams, prompt + a.steps)
    g = torch.Generator(device="cuda").manual_seed(1)
    prompts = torch.randint(3, model.vocab, (a.batch, prompt), generator=g, device="cuda").int()
    beam_decode(model, prompts, a.beams, min(a.steps, 2), eos)  # (first calls load kernels)
    torch.cuda.synchronize()
    t = time.perf_counter()
    hist, scores, _ = beam_decode(model, prompts, a.beams, a.steps, eos)
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    again = rescore(model, hist.view(a.batch * a.beams, -1), prompt, eos).view(a.batch, a.beams)
    for b in range(a.batch):
        print(f"request {b}: {hist[b, 0, prompt:].tolist()} score {scores[b, 0].item():.4f}, fed again "
              f"{again[b, 0].item():.4f}")
    print(f"{a.batch} x {a.beams} beams, {a.steps} steps: {t / a.steps * 1e3:.2f} ms a step")


if __name__ == "__main__":
    with torch.cuda.stream(torch.cuda.Stream()):
        main()

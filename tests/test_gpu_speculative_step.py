"""A speculative decoding step as its operators are used together: drafts drawn by
the sampler from a small 4-bit head, the rows of all drafts through a 4-bit expert
layer and a 4-bit output head, and their verification against the target's
probabilities; eagerly and as one captured graph, whose replays take the device's
own tokens further."""
import numpy as np
import pytest
import torch

from hi_amd import sampler as S
from hi_amd.mx4 import Mx4Experts, Mx4Linear, mx4_rows, quantize_mx4
from hi_amd.speculative import SpecVerifier
from oracle import mx4_oracle, spec_sampled_oracle

pytestmark = pytest.mark.gpu

B, K, V, H, I, E, TOP = 6, 3, 1000, 128, 64, 8, 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Model:
    """One layer for every token: an embedding, experts, a head; the draft model
    is the embedding and a head of its own."""

    def __init__(self, seed):
        g = gen(seed)
        self.embed = torch.randn(V, H, generator=g, device="cuda").bfloat16()
        self.route = torch.randn(H, E, generator=g, device="cuda")
        up = quantize_mx4(torch.randn(E * 2 * I, H, generator=g, device="cuda") * H ** -0.5)
        down = quantize_mx4(torch.randn(E * H, I, generator=g, device="cuda") * I ** -0.5)
        self.experts = Mx4Experts(up[0].view(E, 2 * I, -1), up[1].view(E, 2 * I, -1), down[0].view(E, H, -1),
                                  down[1].view(E, H, -1), max_tokens=B * (K + 1), top_k=TOP)
        head = torch.randn(V, H, generator=g, device="cuda") * 3 * H ** -0.5
        self.head_w = quantize_mx4(head)
        self.head = Mx4Linear(*self.head_w)
        self.draft_head = Mx4Linear(*quantize_mx4(head + 0.3 * torch.randn(V, H, generator=g, device="cuda") * H ** -0.5))
        self.sampler = S.Sampler(B, V, 0, device="cuda")
        self.verifier = SpecVerifier(B, K, V)
        self.params = S.params_to_device(S.row_params(B, temperature=1.0), "cuda")

    def target(self, tokens):
        """Rows of tokens [B][K + 1] -> hidden states, probabilities."""
        x = self.embed[tokens.view(-1).long()]
        w, ids = torch.softmax(x.float() @ self.route, 1).topk(TOP, 1)
        y = x + self.experts(x, ids.int().contiguous(), (w / w.sum(1, keepdim=True)).contiguous())
        logits = self.head(mx4_rows(y))
        return y, logits, torch.softmax(logits, 1).view(B, K + 1, V)

    def step(self, last, draft_u, u):
        """last int32 [B] -> everything the step made, and the next last tokens."""
        tokens, q, t = [last], [], last
        for i in range(K):
            logits = self.draft_head(self.embed[t.long()])
            q.append(torch.softmax(logits, 1))
            t = self.sampler.sample(logits, self.params, draft_u[i])["tokens"]
            tokens.append(t)
        rows = torch.stack(tokens, 1)
        y, logits, p = self.target(rows)
        q, drafts = torch.stack(q, 1), rows[:, 1:].contiguous()
        out = self.verifier(p, drafts, u, draft_probs=q)
        n = (out["counts"].long() - 1)[:, None]
        return {"y": y, "logits": logits, "p": p, "q": q, "drafts": drafts, "tokens": out["tokens"],
                "counts": out["counts"], "last": out["tokens"].gather(1, n)[:, 0].contiguous()}


def numbers(step):
    g = gen(1000 + step)
    return torch.rand(K, B, generator=g, device="cuda"), torch.rand(B, K + 1, generator=g, device="cuda")


def check(model, got, u):
    """The head's logits from the layer's own states, and the tokens from the
    step's own probabilities."""
    w = mx4_oracle.values(*model.head_w)
    x = mx4_oracle.rounded(got["y"])
    size = x.abs() @ w.abs().t()
    assert ((got["logits"].double().cpu() - x @ w.t()).abs() <= (H // 32 + 8) * 2.0 ** -23 * size).all()
    f64 = lambda t: t.double().cpu().numpy()
    tokens, counts = spec_sampled_oracle.verify(f64(got["p"]), got["drafts"].cpu().numpy(), u.cpu().numpy(), f64(got["q"]))
    assert np.array_equal(got["tokens"].cpu().numpy(), tokens) and np.array_equal(got["counts"].cpu().numpy(), counts)
    return counts


def test_steps(hip):
    model = Model(1)
    last, seen = torch.arange(B, dtype=torch.int32, device="cuda"), set()
    for step in range(8):
        du, u = numbers(step)
        got = model.step(last, du, u)
        seen |= set(check(model, got, u).tolist())
        last = got["last"]
    assert len(seen) >= 3  # some drafts taken, some not


def test_captured_step(hip):
    """One graph of the whole step, replayed on what it emitted itself."""
    model, eager = Model(2), Model(2)
    last = torch.arange(B, dtype=torch.int32, device="cuda")
    du, u = numbers(0)
    model.step(last, du, u)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = model.step(last, du, u)
    begin = last.clone()
    for step in range(5):
        ndu, nu = numbers(step)
        du.copy_(ndu)
        u.copy_(nu)
        last.copy_(begin)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(model, got, u)
        want = eager.step(begin, ndu, nu)
        assert torch.equal(got["tokens"], want["tokens"]) and torch.equal(got["counts"], want["counts"])
        begin = got["last"].clone()

"""Router, experts, 4-bit products, beam selection and state reordering in one
decoder: the hypotheses' scores against the same sequences fed again without
any reordering, and the search against one that keeps a cache per hypothesis by
recomputing it."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("moe_beam_decode", os.path.join(ROOT, "examples", "moe_beam_decode.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(autouse=True)
def stream(hip):
    import torch
    with torch.cuda.stream(torch.cuda.Stream()):
        yield


def _model(example, rows, max_len):
    return example.Decoder(rows, max_len, vocab=1000, hidden=256, heads=4, experts=16, top_k=3, inter=128, group=32)


def _tolerance(scores, steps, lse):
    # Each step rounds lse (and its sum, a few units), l - lse and c + (l - lse)
    # to f32; a score's size is that of the largest partial sum.
    return steps * (abs(scores) * 2.0 ** -24 + lse * 2.0 ** -21)


@pytest.mark.parametrize("batch,beams,steps", [(1, 4, 12), (3, 5, 9), (2, 1, 6)])
def test_scores_of_hypotheses(hip, example, batch, beams, steps):
    import torch
    start, eos = 3, 7
    model = _model(example, batch * beams, start + steps)
    g = torch.Generator(device="cuda").manual_seed(beams)
    prompts = torch.randint(8, 1000, (batch, start), generator=g, device="cuda").int()
    hist, scores, finished = example.beam_decode(model, prompts, beams, steps, eos)
    assert torch.equal(hist[:, :, :start], prompts[:, None].expand(-1, beams, -1))
    assert (scores[:, :-1] >= scores[:, 1:]).all()
    assert torch.equal(finished.bool(), (hist[:, :, start:] == eos).any(2))
    for b in range(batch):
        assert len({tuple(h) for h in hist[b].tolist()}) == beams
    again = example.rescore(model, hist.reshape(batch * beams, -1), start, eos).view(batch, beams)
    for got, want in zip(scores.view(-1).tolist(), again.view(-1).tolist()):
        assert abs(got - want) <= _tolerance(want, steps, 16.0)


def test_search_against_recomputation(hip, example):
    """Each step's candidates by feeding every hypothesis from its start."""
    import torch
    batch, beams, steps, start, eos = 2, 3, 6, 3, 7
    rows = batch * beams
    model = _model(example, rows, start + steps)
    g = torch.Generator(device="cuda").manual_seed(11)
    prompts = torch.randint(8, 1000, (batch, start), generator=g, device="cuda").int()
    hist, scores, _ = example.beam_decode(model, prompts, beams, steps, eos)
    kept = [[(prompts[b].tolist(), 0.0)] for b in range(batch)]
    for i in range(steps):
        feed = [kept[b][j % len(kept[b])][0] for b in range(batch) for j in range(beams)]
        seq = torch.tensor(feed, dtype=torch.int32, device="cuda")
        for at in range(start + i):
            logits = model.step(seq[:, at], at)
        logp = torch.log_softmax(logits.double(), 1).cpu()
        for b in range(batch):
            found = []
            for j, (h, c) in enumerate(kept[b]):
                if eos in h[start:]:
                    found.append((c, h + [eos]))
                    continue
                top = logp[b * beams + j].topk(beams)
                found += [(c + v, h + [t]) for v, t in zip(top.values.tolist(), top.indices.tolist())]
            found.sort(key=lambda x: -x[0])
            # decided by more than the f32 scores may be off by
            gap = min(x[0] - y[0] for x, y in zip(found[:beams], found[1:beams + 1]))
            assert gap > 2 * _tolerance(found[0][0], steps, 16.0), "a tie: take another seed"
            kept[b] = [(h, c) for c, h in found[:beams]]
    assert hist.tolist() == [[h for h, _ in kept[b]] for b in range(batch)]
    for b in range(batch):
        for got, (_, want) in zip(scores[b].tolist(), kept[b]):
            assert abs(got - want) <= _tolerance(want, steps, 16.0)

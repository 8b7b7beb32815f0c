"""Whose memory an operator with buffers of its own takes: the given stream's,
as its work there is ordered behind what the memory held before, and the
allocator gives it back in that stream's order.  On the CPU, by an allocator
that notes the stream; on the GPU, beside a stream that is busy."""
import contextlib
import types

import pytest
import torch

from hi_amd import beam, moe, mx4, sampler
from hi_amd.mx4 import Mx4Experts, Mx4Linear, quantize_mx4
from hi_amd.speculative import SpecVerifier
from oracle import spec_sampled_oracle

SIDE = types.SimpleNamespace(name="side")


@pytest.fixture
def allocations(monkeypatch):
    """The stream (None: the current one) of every torch.empty and torch.zeros."""
    at, made = [None], []

    @contextlib.contextmanager
    def on(stream):
        at.append(stream)
        yield
        at.pop()

    def noting(fn):
        def new(*a, **kw):
            made.append(at[-1])
            return fn(*a, **kw)
        return new

    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch, "empty", noting(torch.empty))
    monkeypatch.setattr(torch, "zeros", noting(torch.zeros))
    return made


def _codes(*shape):
    return torch.full((*shape[:-1], shape[-1] // 2), 1, dtype=torch.uint8), torch.full(
        (*shape[:-1], shape[-1] // 32), 127, dtype=torch.uint8)


@pytest.mark.parametrize("stream", [None, SIDE])
def test_experts_buffers(monkeypatch, allocations, stream):
    monkeypatch.setattr(mx4, "_on", lambda *a: None)
    monkeypatch.setattr(mx4, "_pack", lambda *a: beam._empty((16,), torch.uint8, "cpu", a[-1]))
    layer = Mx4Experts(*_codes(3, 128, 96), *_codes(3, 96, 64), max_tokens=5, top_k=2, stream=stream)
    # weights twice, rows, activations, terms, the groups' three
    assert allocations == [stream] * 8
    assert layer._y.shape == (10, 96) and layer._groups.order.numel() == 10


@pytest.mark.parametrize("stream", [None, SIDE])
def test_beam_and_bf16_experts_buffers(monkeypatch, allocations, stream):
    beam.BeamSearch(2, 4, 1000, device="cpu", stream=stream)
    monkeypatch.setattr(moe, "_on", lambda *a: None)
    moe.MoeExperts(torch.ones(3, 128, 96).bfloat16(), torch.ones(3, 96, 64).bfloat16(), 5, 2, stream=stream)
    assert allocations == [stream] * 6


@pytest.mark.parametrize("stream", [None, SIDE])
def test_sampler_outputs(monkeypatch, allocations, stream):
    monkeypatch.setattr(sampler, "_zeroed", lambda *a: beam._empty((16,), torch.uint8, "cpu", a[-1]))
    monkeypatch.setattr(sampler, "_stream_ptr", lambda s: 0)
    one = sampler.Sampler(2, 50, n_logprobs=3, stream=stream)
    monkeypatch.setattr(sampler, "load", lambda: types.SimpleNamespace(hi_rocm_sample=lambda *a: 0))
    x = torch.ones(2, 50)
    out = one.sample(x, x, x, n_logprobs=3, token_logprobs=True, stream=stream)
    assert allocations == [stream] * 5 and out["logprob_ids"].shape == (2, 3)


@pytest.mark.parametrize("make", [lambda **kw: SpecVerifier(4, 2, 1000, **kw), lambda **kw: sampler.Sampler(4, 1000, **kw)],
                         ids=["verifier", "sampler"])
@pytest.mark.parametrize("capturing", [False, True])
@pytest.mark.parametrize("stream", [None, "side"])
def test_zeroed_workspace(monkeypatch, make, stream, capturing):
    """Zeroed on the given stream, and waited for there: a first call on any other
    finds the zeros.  (A capture cannot wait, and orders the fill itself.)"""
    done, at = [], []

    class Stream:
        device_index = 0

        def __init__(self, name):
            self.name = name

        def synchronize(self):
            done.append(("waited", self.name))

    class Zeros:
        device = torch.device("cuda:0")

        def get_device(self):
            return 0

    def zeros(*a, **kw):
        done.append(("filled", at[-1].name if at else "current"))
        return Zeros()

    @contextlib.contextmanager
    def on(s):
        at.append(s)
        yield
        at.pop()

    monkeypatch.setattr(torch, "zeros", zeros)
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream("current"))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    make(**({"stream": Stream("side")} if stream else {}))
    name = stream or "current"
    assert done == [("filled", name)] + [("waited", name)] * (not capturing)
    if stream:
        elsewhere = Stream("elsewhere")
        elsewhere.device_index = 1
        with pytest.raises(ValueError, match="cuda:1"):
            make(stream=elsewhere)


def _busy(x, ms):
    """Some milliseconds of work on the current stream."""
    y = x @ x
    for _ in range(ms):
        y = x @ y
    return y


@pytest.mark.gpu
def test_layer_of_a_side_stream(hip, new_stream):
    """Made and called on a stream while the current one is busy with memory that it
    has given back: the results of the same layer alone."""
    g = torch.Generator(device="cuda").manual_seed(1)
    E, H, I, T, K = 6, 256, 96, 300, 2
    up = quantize_mx4(torch.randn(E * 2 * I, H, generator=g, device="cuda") * H ** -0.5)
    down = quantize_mx4(torch.randn(E * H, I, generator=g, device="cuda") * I ** -0.5)
    args = (up[0].view(E, 2 * I, -1), up[1].view(E, 2 * I, -1), down[0].view(E, H, -1), down[1].view(E, H, -1))
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    ids = torch.rand(T, E, generator=g, device="cuda").topk(K, 1).indices.int()
    wts = torch.rand(T, K, generator=g, device="cuda")
    want = Mx4Experts(*args, max_tokens=T, top_k=K)(x, ids, wts)
    a = torch.randn(4096, 4096, generator=g, device="cuda").bfloat16()
    side = new_stream()
    torch.cuda.synchronize()
    for size in (T * K * H, T * H, E * 2 * I * H):
        _busy(a, 4)
        late = torch.empty(size, device="cuda")
        late.fill_(float("nan"))  # (runs behind the products, in memory that is free at once)
        del late
    got = Mx4Experts(*args, max_tokens=T, top_k=K, stream=side)(x, ids, wts, stream=side)
    lin = Mx4Linear(*up, stream=side)(x, stream=side)
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert torch.equal(lin, Mx4Linear(*up)(x))


@pytest.mark.gpu
def test_verifier_on_another_stream(hip, new_stream):
    """A verifier made while the current stream is busy, called on another at once."""
    g = torch.Generator(device="cuda").manual_seed(2)
    B, K, V = 5, 3, 9000
    p = torch.softmax(torch.randn(B, K + 1, V, generator=g, device="cuda") * 2, 2)
    q = torch.softmax(torch.randn(B, K, V, generator=g, device="cuda") * 2, 2)
    t = torch.randint(0, V, (B, K), generator=g, device="cuda").int()
    u = torch.rand(B, K + 1, generator=g, device="cuda")
    a = torch.randn(4096, 4096, generator=g, device="cuda").bfloat16()
    side, own = new_stream(), new_stream()
    f64 = lambda x: x.double().cpu().numpy()
    want, counts = spec_sampled_oracle.verify(f64(p), t.cpu().numpy(), u.cpu().numpy(), f64(q))
    torch.cuda.synchronize()
    for kw in ({}, {"stream": own}):
        _busy(a, 8)
        verifier = SpecVerifier(B, K, V, **kw)
        for _ in range(3):
            out = verifier(p, t, u, draft_probs=q, stream=side)
            side.synchronize()
            assert (out["tokens"].cpu().numpy() == want).all() and (out["counts"].cpu().numpy() == counts).all()
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_verifier_made_in_a_capture(hip):
    """The fill is the graph's then: every replay begins with a workspace of zeros."""
    g = torch.Generator(device="cuda").manual_seed(3)
    B, K, V = 3, 2, 20000
    p = torch.softmax(torch.randn(B, K + 1, V, generator=g, device="cuda") * 2, 2)
    t = torch.randint(0, V, (B, K), generator=g, device="cuda").int()
    u = torch.rand(B, K + 1, generator=g, device="cuda")
    eager = SpecVerifier(B, K, V)
    eager(p, t, u)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        verifier = SpecVerifier(B, K, V)
        out = verifier(p, t, u)
    for i in range(4):
        p.copy_(torch.softmax(torch.randn(B, K + 1, V, generator=g, device="cuda") * 2, 2))
        u.copy_(torch.rand(B, K + 1, generator=g, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = eager(p, t, u)
        assert torch.equal(out["tokens"], want["tokens"]) and torch.equal(out["counts"], want["counts"])


@pytest.mark.gpu
def test_sampler_on_another_stream(hip, new_stream):
    """As above for the sampler, whose workspace begins as zeros too."""
    g = torch.Generator(device="cuda").manual_seed(4)
    B, V = 6, 50000
    x, u = torch.randn(B, V, generator=g, device="cuda") * 3, torch.rand(B, generator=g, device="cuda")
    params = sampler.params_to_device(sampler.row_params(B, temperature=0.8, top_p=0.9), "cuda")
    a = torch.randn(4096, 4096, generator=g, device="cuda").bfloat16()
    side, own = new_stream(), new_stream()
    want = sampler.Sampler(B, V).sample(x, params, u)["tokens"].clone()
    torch.cuda.synchronize()
    for kw in ({}, {"stream": own}):
        _busy(a, 8)
        one = sampler.Sampler(B, V, **kw)
        for _ in range(3):
            got = one.sample(x, params, u, stream=side)["tokens"]
            side.synchronize()
            assert torch.equal(got, want)
        torch.cuda.synchronize()

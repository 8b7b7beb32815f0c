"""Verification of sampled drafts against the rule in 64 bits: tokens and counts
are equal.  (The kernel's f64 sums are off by some V 2^-53 of the total, so a
random number would have to lie that near to a border to tell them apart.)"""
import numpy as np
import pytest
import torch

from hi_amd import _lib
from hi_amd.speculative import SpecVerifier
from oracle import spec_sampled_oracle as O

pytestmark = pytest.mark.gpu


def make(B, K, V, dtype, draft, seed, sharp=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, K + 1, V, generator=g) * sharp
    p = torch.softmax(x, 2).to(dtype)
    y = x[:, :K] + torch.randn(B, K, V, generator=g)
    q = torch.softmax(y, 2)
    tokens = (q.reshape(-1, V).multinomial(1, generator=g).view(B, K) if K else torch.zeros(B, 0)).int()
    u = torch.rand(B, K + 1, generator=g)
    return p, (q.to(dtype) if draft else None), tokens, u


def check(p, q, tokens, u, lengths=None, plan=None, **kw):
    B, K, V = p.shape[0], p.shape[1] - 1, p.shape[2]
    plan = plan or SpecVerifier(B, K, V)
    dev = lambda t: None if t is None else t if t.is_cuda else t.cuda()
    out = plan(dev(p), dev(tokens), dev(u), draft_probs=dev(q), draft_len=dev(lengths), **kw)
    f64 = lambda t: None if t is None else t.double().cpu().numpy()
    want, counts = O.verify(f64(p), tokens.cpu().numpy(), u.cpu().numpy(), f64(q),
                            None if lengths is None else lengths.cpu().numpy())
    torch.cuda.synchronize()
    assert np.array_equal(out["counts"].cpu().numpy(), counts)
    assert np.array_equal(out["tokens"].cpu().numpy().reshape(want.shape), want)
    return want, counts


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("B,K,V", [(1, 0, 1), (1, 1, 1), (3, 2, 2), (2, 4, 7), (5, 3, 63), (4, 1, 257), (2, 3, 4099),
                                   (7, 5, 1000), (3, 70, 129), (1, 4, 20001), (2, 2, 100000)])
def test_rule(hip, dtype, draft, B, K, V):
    check(*make(B, K, V, dtype, draft, seed=B + K + V))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_requests(hip, dtype):
    """Long parts (many requests of a large vocabulary) and short ones."""
    for B, V in ((40, 128256), (300, 999), (70, 50257)):
        lengths = torch.randint(-2, 6, (B,), generator=torch.Generator().manual_seed(B)).int()
        want, counts = check(*make(B, 3, V, dtype, True, seed=B, sharp=1.0), lengths=lengths)
        assert len(np.unique(counts)) >= 3


def test_random_numbers_at_their_ends(hip):
    """0 and the largest below 1: drafts of probability 0 are never accepted,
    others always at 0; the draw takes the first and the last token with mass."""
    p, q, t, u = make(64, 4, 300, torch.float32, True, seed=3)
    p[:, :, :5] = 0.0
    p[:, :, 295:] = 0.0
    for value in (0.0, 1.0 - 2.0 ** -24):
        want, counts = check(p, q, t, torch.full_like(u, value))
        for b in range(64):
            assert 5 <= want[b, counts[b] - 1] < 295
    t[:, 2] = 2  # no mass
    want, counts = check(p, q, t, torch.zeros_like(u))
    assert (counts <= 3).all()


def test_drafts_that_are_no_token(hip):
    for bad in (-1, 300, 2 ** 31 - 1):
        for draft in (True, False):
            p, q, t, u = make(6, 3, 300, torch.float32, draft, seed=4)
            t[:, 1] = bad
            want, counts = check(p, q, t, u)
            assert (counts <= 2).all() and (want[:, :2] >= -1).all()


def test_nothing_left(hip):
    """Rows without mass: p = q after a draft of probability 0 (the token comes
    from p), p all 0 (token 0), over more than one part of a row."""
    for V in (64, 30000):
        p, q, t, u = make(4, 2, V, torch.float32, True, seed=V)
        p[:, :, V // 2] = 0.0
        q[:] = p[:, :2]
        t[:, 0] = V // 2  # never accepted, and nothing is left
        check(p, q, t, u)
        p[1:3] = 0.0
        want, _ = check(p, q, t, u)
        assert (want[1:3, 0] == 0).all()
        p[0, 0, 5:V // 2] = -1.0
        check(p, q, t, u)


def test_nan_and_equal_rows(hip):
    """NaN in p or q leaves its token out; drafts at u q = p are rejected."""
    p, q, t, u = make(8, 3, 500, torch.float32, True, seed=9)
    p[0, :, 7] = float("nan")
    q[1, :, 8] = float("nan")
    p[2] = float("nan")
    t[3, 0], q[3, 0, int(t[3, 0])], p[3, 0, int(t[3, 0])], u[3, 0] = 11, 0.5, 0.25, 0.5
    q[3, 0, 11], p[3, 0, 11] = 0.5, 0.25
    want, counts = check(p, q, t, u)
    assert counts[3] == 1 and counts[2] == 1 and want[2, 0] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(hip, dtype):
    """Views of larger tensors, rows that start anywhere, one row for all."""
    B, K, V = 3, 2, 333
    p, q, t, u = make(B, K, V, dtype, True, seed=12)
    for off in range(1, 4):
        big = torch.full((B, K + 2, V + 10 + off), float("nan"), dtype=dtype, device="cuda")
        bigq = torch.full((B, K + 1, V + 7), float("nan"), dtype=dtype, device="cuda")
        vp, vq = big[:, :K + 1, off:off + V], bigq[:, :K, 3:3 + V]
        vp.copy_(p)
        vq.copy_(q)
        check(vp, vq, t, u)
    one = p[:1, :1].cuda().expand(B, K + 1, V)
    check(one, q, t, u)


def test_rows_far_apart(hip):
    """Requests whose offsets pass 32 bits, in values and in bytes."""
    B, K, V = 3, 2, 5000
    p, q, t, u = make(B, K, V, torch.float32, True, seed=21)
    far = 2 ** 31 + 12
    place = torch.empty((B - 1) * far + (K + 1) * 6000, device="cuda")
    vp = place.as_strided((B, K + 1, V), (far, 6000, 1))
    vp.copy_(p)
    check(vp, q, t, u)


def test_workspace_serves_any_batch(hip):
    """Large and small batches in turn, types mixed: the counters stay ready."""
    plan = SpecVerifier(64, 3, 40000)
    for i, B in enumerate((64, 1, 33, 2, 64, 5)):
        dtype = (torch.float32, torch.bfloat16)[i % 2]
        check(*make(B, 3, 40000, dtype, i % 3 != 0, seed=i), plan=plan)
    assert not plan.workspace[:plan.workspace.numel() // 2].any()  # the counters' half


def test_frequencies(hip):
    """Emitted first tokens follow p whatever q is: 200,000 requests of a
    vocabulary of 8, each count within 5 standard deviations."""
    B, V, rounds = 50000, 8, 4
    g = torch.Generator(device="cuda").manual_seed(77)
    p = torch.softmax(torch.randn(V, generator=g, device="cuda"), 0)
    q = torch.softmax(torch.randn(V, generator=g, device="cuda"), 0)
    plan = SpecVerifier(B, 1, V)
    hits = torch.zeros(V, dtype=torch.long, device="cuda")
    for _ in range(rounds):
        t = torch.multinomial(q, B, replacement=True, generator=g).int().view(B, 1)
        u = torch.rand(B, 2, generator=g, device="cuda")
        out = plan(p.expand(B, 2, V), t, u, draft_probs=q.expand(B, 1, V))
        hits += torch.bincount(out["tokens"][:, 0].long(), minlength=V)
    n = B * rounds
    dev = (hits.double() / n - p.double()).abs() / (p.double() * (1 - p.double()) / n).sqrt()
    assert (dev < 5).all(), dev


def test_graph_and_streams(hip, new_stream):
    """A captured call replays on new inputs, beside eager calls on another
    stream with a workspace of their own."""
    plan, other = SpecVerifier(6, 3, 9000), SpecVerifier(6, 3, 9000)
    sets = [make(6, 3, 9000, torch.float32, True, seed=s) for s in range(4)]
    bufs = [t.cuda() for t in sets[0]]
    out = plan.outputs(6)
    side = new_stream()
    plan(bufs[0], bufs[2], bufs[3], draft_probs=bufs[1], out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan(bufs[0], bufs[2], bufs[3], draft_probs=bufs[1], out=out)
    for s in sets[1:] + sets[:1]:
        for dst, src in zip(bufs, s):
            dst.copy_(src)
        torch.cuda.synchronize()
        graph.replay()
        got = other(bufs[0], bufs[2], bufs[3], draft_probs=bufs[1], stream=side)
        torch.cuda.synchronize()
        want, counts = O.verify(s[0].double().numpy(), s[2].numpy(), s[3].numpy(), s[1].double().numpy())
        for o in (out, got):
            assert np.array_equal(o["tokens"].cpu().numpy(), want) and np.array_equal(o["counts"].cpu().numpy(), counts)


def test_refused(hip):
    p, q, t, u = (x.cuda() for x in make(2, 2, 50, torch.float32, True, seed=1))
    plan = SpecVerifier(2, 2, 50)
    calls = [dict(target_probs=p.half()), dict(target_probs=p[:, :2]), dict(target_probs=p.transpose(0, 1)),
             dict(target_probs=torch.cat((p, p))), dict(draft_probs=q.bfloat16()), dict(draft_probs=q[:, :1]),
             dict(draft_tokens=t.long()), dict(draft_tokens=t[:, :1]), dict(uniforms=u.double()), dict(uniforms=u[:, :2]),
             dict(draft_len=torch.ones(3, dtype=torch.int32, device="cuda")), dict(draft_tokens=t.cpu()),
             dict(target_probs=torch.zeros(2, 3, 100, device="cuda")[:, :, ::2])]
    for changed in calls:
        args = dict(target_probs=p, draft_tokens=t, uniforms=u, draft_probs=q)
        args.update(changed)
        with pytest.raises(ValueError):
            plan(**args)
    with pytest.raises(ValueError):
        SpecVerifier(2, -1, 50)
    with pytest.raises(_lib.HiRocmError):
        SpecVerifier(70000, 2, 50)

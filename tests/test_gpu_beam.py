"""Beam selection and state reordering against the definitions in 64 bits.

A score is three f32 roundings (lse, l - lse, + c) beside lse's own error:
the sum of up to 64 terms a thread, a tree over the workgroup and the row's
parts, each term's exponential within a few units of its last place, and a
logarithm.  SUM_EPS bounds that sum's relative error, which is lse's absolute
one."""
import math

import numpy as np
import pytest
import torch

from hi_amd import _lib
from hi_amd.beam import BeamSearch, reorder_states

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
SUM_EPS = (64 + 6 + 4 + 16 + 6 + 8) * EPS


def definition(x, c, finished, eos, mask, K, n):
    """All candidates of each request: (score64, beam, logit, token), in the
    order (score, beam, logit, token) of the exact scores, and the tolerance."""
    x = x.astype(np.float64)
    out, tol = [], 0.0
    for b in range(x.shape[0] // K):
        cand = []
        for k in range(K):
            r = b * K + k
            if not np.isfinite(c[r]):
                continue
            if finished is not None and finished[r]:
                cand.append((float(c[r]), k, 0.0, eos))
                continue
            l = x[r].copy()
            l[np.isnan(l)] = -np.inf
            if mask is not None:
                l[~mask[r]] = -np.inf
            m = l.max()
            if not np.isfinite(m):
                continue
            lse = m + math.log(np.exp(l - m).sum())
            ids = np.nonzero(l > -np.inf)[0]
            ids = ids[np.lexsort((ids, -l[ids]))][:n]
            s = float(c[r]) + (l[ids] - lse)
            tol = max(tol, EPS * (4 * abs(lse) + 2 * np.abs(l[ids] - lse).max() + 2 * np.abs(s).max()) + SUM_EPS)
            cand += [(float(v), k, float(l[i]), int(i)) for v, i in zip(s, ids)]
        out.append(sorted(cand, key=lambda t: (-t[0], t[1], -t[2], t[3])))
    return out, tol


def check(res, want, tol, K, n, eos, finished):
    s, t, p, f = (res[k].cpu().numpy() for k in ("scores", "tokens", "parents", "finished"))
    for b, cand in enumerate(want):
        have = min(n, len(cand))
        exact = {(k, i): (v, l, rank) for rank, (v, k, l, i) in enumerate(cand)}
        seen = {}
        for j in range(have):
            key = (int(p[b, j]), int(t[b, j]))
            assert key in exact, (b, j, key)  # a candidate of its beam's first n
            v, l, _ = exact[key]
            assert abs(s[b, j] - v) <= tol, (b, j, s[b, j], v, tol)
            assert abs(s[b, j] - cand[j][0]) <= tol, (b, j)  # the j-th best score
            if j:  # scores descend, the lower beam first on equal ones
                assert s[b, j] < s[b, j - 1] or (s[b, j] == s[b, j - 1] and p[b, j] >= p[b, j - 1]), (b, j)
            seen.setdefault(key[0], []).append(key)
            done = finished is not None and bool(finished[b * K + key[0]])
            assert f[b, j] == (done or key[1] == eos)
        for k, keys in seen.items():  # within a beam: the first ones, in the logits' order
            order = [(kk, i) for _, kk, _, i in sorted((c for c in cand if c[1] == k), key=lambda c: (-c[2], c[3]))]
            assert keys == order[:len(keys)], (b, k)
        for j in range(have, n):
            assert s[b, j] == -np.inf and t[b, j] == (0 if eos is None else eos) and p[b, j] == j % K and f[b, j] == 1


def run(x, c, K, n, finished=None, eos=None, mask=None, bs=None, stream=None):
    dev = "cuda"
    B, V = x.shape[0] // K, x.shape[1]
    words = None
    if mask is not None:
        pad = np.zeros((x.shape[0], (V + 31) // 32 * 32), bool)
        pad[:, :V] = mask.cpu().numpy() if torch.is_tensor(mask) else mask
        words = torch.from_numpy(np.packbits(pad, axis=1, bitorder="little").view(np.int32).copy()).to(dev)
    bs = bs or BeamSearch(B, K, V, n)
    fin = None if finished is None else torch.from_numpy(np.asarray(finished, np.uint8)).to(dev)
    res = bs.select(x, torch.from_numpy(np.asarray(c, np.float32)).to(dev), finished=fin, eos_id=eos, mask_words=words,
                    stream=stream)
    torch.cuda.synchronize()
    return res


def agree(x, c, K, n, finished=None, eos=None, mask=None, **kw):
    res = run(x, c, K, n, finished, eos, mask, **kw)
    want, tol = definition(x.float().cpu().numpy(), np.asarray(c, np.float32), finished, eos, mask, K, n)
    check(res, want, tol, K, n, eos, finished)
    return res


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,n", [(1, 1, 1, 1), (1, 1, 2, 4), (2, 3, 17, 6), (1, 4, 5003, 8), (3, 2, 4096, 64),
                                     (1, 32, 777, 64), (2, 5, 50257, 5), (7, 4, 16381, 8), (40, 8, 33000, 16)])
def test_selection(hip, dtype, B, K, V, n):
    g = torch.Generator(device="cuda").manual_seed(B * 1000 + V)
    x = (torch.randn(B * K, V, generator=g, device="cuda") * 2.5).to(dtype)
    c = -30.0 * np.random.default_rng(V).random(B * K)
    fin = np.random.default_rng(K).random(B * K) < 0.25
    agree(x, c, K, n)
    agree(x, c, K, n, finished=fin, eos=V // 2)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("offset", range(8))
def test_rows_at_any_alignment(hip, dtype, offset):
    g = torch.Generator(device="cuda").manual_seed(offset)
    K, V, n = 3, 4099, 6
    big = (torch.randn(K * 4, V + 13, generator=g, device="cuda") * 3).to(dtype)
    x = big[:, offset:offset + V]
    agree(x, [-1.0 * i for i in range(K * 4)], K, n)


def test_masks(hip):
    """A fifth of the tokens, a single one, none, and all but one part."""
    rng = np.random.default_rng(3)
    K, V, n = 4, 20011, 8
    x = torch.from_numpy(rng.standard_normal((8, V)).astype(np.float32) * 3).cuda()
    mask = rng.random((8, V)) < 0.2
    mask[1] = False
    mask[2] = False
    mask[2, V - 1] = True
    mask[3] = False
    mask[3, :5] = True
    mask[5] = False
    mask[6] = False
    mask[7] = False
    mask[4] = False
    agree(x, -rng.random(8) * 5, K, n, mask=mask, eos=7)  # the second request has no candidate at all


def test_special_logits(hip):
    rng = np.random.default_rng(4)
    K, V, n = 6, 9001, 12
    x = rng.standard_normal((2 * K, V)).astype(np.float32)
    x[0, 10:20] = np.nan
    x[0, 0] = np.nan
    x[1] = np.nan                       # no candidate
    x[2, 5] = np.inf                    # none either: every other probability is 0
    x[3] = -np.inf
    x[3, 77] = 1.0                      # one candidate of probability 1
    x[4] = np.finfo(np.float32).min     # lowest value everywhere: V equal candidates
    x[5, ::2] = -np.inf
    x[6, :] = 0.0
    x[6, 1::2] = -0.0                   # equal to 0: the lower token first
    x[7, 100] = np.finfo(np.float32).max
    c = np.array([-1, -2, -3, -4, -5, -6, -1, -2, -np.inf, np.nan, np.inf, -3], np.float32)
    agree(torch.from_numpy(x).cuda(), c, K, n)


@pytest.mark.parametrize("levels", [1, 2, 40])
@pytest.mark.parametrize("V", [300, 20000, 70000])
def test_many_equal_logits(hip, levels, V):
    rng = np.random.default_rng(levels)
    x = rng.integers(0, levels, (6, V)).astype(np.float32)
    agree(torch.from_numpy(x).cuda(), [0.0] * 6, 3, 33)
    agree(torch.from_numpy(x).cuda().bfloat16(), [0.0, -1e6, 0.0, 0.0, 0.0, 0.0], 3, 64)


def test_equal_scores_of_beams(hip):
    """Beams that agree in everything: the lower beam first, at every rank."""
    rng = np.random.default_rng(6)
    row = rng.standard_normal(3000).astype(np.float32)
    res = agree(torch.from_numpy(np.stack([row] * 8)).cuda(), [-2.0] * 8, 8, 24)
    assert res["parents"].cpu().tolist()[0] == list(range(8)) * 3
    fin = [1] * 8
    res = agree(torch.from_numpy(np.stack([row] * 8)).cuda(), [-2.0] * 8, 8, 8, finished=fin, eos=5)
    assert res["parents"].cpu().tolist()[0] == list(range(8)) and res["tokens"].unique().tolist() == [5]


def test_long_rows_and_workspace_reuse(hip):
    """A vocabulary of many parts; one workspace for batches of other sizes."""
    rng = np.random.default_rng(8)
    V, K = 600001, 2
    bs = BeamSearch(9, K, V, 8)
    for B in (1, 9, 2):
        x = torch.from_numpy(rng.standard_normal((B * K, V)).astype(np.float32)).cuda()
        agree(x, -rng.random(B * K), K, 8, bs=bs)


def test_same_bits_every_time_and_on_streams(hip):
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(64, 30000, generator=g, device="cuda").bfloat16()
    torch.cuda.synchronize()
    first = run(x, np.linspace(-9, 0, 64), 8, 16)
    for _ in range(3):
        again = run(x, np.linspace(-9, 0, 64), 8, 16, stream=torch.cuda.Stream())
        for k in first:
            assert torch.equal(first[k], again[k]), k


def test_selection_in_a_graph(hip):
    g = torch.Generator(device="cuda").manual_seed(10)
    K, V, n = 4, 12345, 8
    bs = BeamSearch(2, K, V, n)
    x = torch.randn(2 * K, V, generator=g, device="cuda")
    c = torch.zeros(2 * K, device="cuda")
    out = bs.outputs(2)
    bs.select(x, c, out=out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        bs.select(x, c, out=out)
    for i in range(4):
        x.copy_(torch.randn(2 * K, V, generator=g, device="cuda") * (i + 1))
        c.copy_(-torch.rand(2 * K, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = {k: v.clone() for k, v in out.items()}
        want = run(x, c.cpu().numpy(), K, n)
        for k in got:
            assert torch.equal(got[k], want[k]), (i, k)


# ---- states ---------------------------------------------------------------

def moved(src, dst, parents, row_dim, length_dim=None, lengths=None):
    """The definition, a row at a time."""
    B, K = parents.shape
    s, d = src.movedim(row_dim, 0), dst.movedim(row_dim, 0).clone()
    for b in range(B):
        for j in range(K):
            p = int(parents[b, j])
            p = p if 0 <= p < K else j
            a, t = s[b * K + p], d[b * K + j]
            if lengths is None:
                t.copy_(a)
            else:
                at = length_dim - 1
                n = max(0, min(int(lengths[b]), a.shape[at]))
                t.narrow(at, 0, n).copy_(a.narrow(at, 0, n))
    return d.movedim(0, row_dim)


LAYOUTS = [((6, 5), 0, None), ((2, 6, 3, 7, 16), 1, 3), ((6, 9, 8), 0, 1), ((3, 2, 6, 5, 2, 24), 2, 4), ((6,), 0, None),
           ((4, 6, 3), 1, None), ((6, 2, 11, 3), 0, 2), ((2, 6, 1, 40, 1, 128), 1, 3)]


@pytest.mark.parametrize("shape,row_dim,length_dim", LAYOUTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8, torch.int32])
@pytest.mark.parametrize("place", ["other", "in place"])
def test_reorder(hip, shape, row_dim, length_dim, dtype, place):
    rng = np.random.default_rng(len(shape))
    src = torch.from_numpy(rng.integers(0, 250, shape)).to(dtype).cuda()
    for parents in ([[0, 1, 2], [2, 0, 0]], [[2, 2, 2], [1, 2, 0]], [[0, 1, 2], [0, 1, 2]], [[-1, 3, 1], [2, 1, 99]]):
        par = torch.tensor(parents, dtype=torch.int32, device="cuda")
        lens = None
        if length_dim is not None:
            lens = torch.tensor([rng.integers(0, shape[length_dim] + 1), shape[length_dim] + 5], dtype=torch.int32,
                                device="cuda")
        dst = src.clone() if place == "in place" else torch.full_like(src, 7)
        want = moved(src, dst, par.cpu(), row_dim, length_dim, None if lens is None else lens.cpu())
        if place == "in place":
            got = reorder_states(dst, par, row_dim=row_dim, length_dim=length_dim, lengths=lens)
            assert got is dst
        else:
            got = reorder_states(src, par, dst=dst, row_dim=row_dim, length_dim=length_dim, lengths=lens)
        torch.cuda.synchronize()
        assert torch.equal(got.cpu(), want.cpu())


@pytest.mark.parametrize("beams", [1, 2, 4, 5, 8, 9, 16, 17, 32])
def test_reorder_beams(hip, beams):
    g = torch.Generator(device="cuda").manual_seed(beams)
    src = torch.randn(3, 4 * beams, 2, 33, 8, generator=g, device="cuda").bfloat16()
    par = torch.randint(0, beams, (4, beams), generator=g, device="cuda").int()
    lens = torch.tensor([33, 0, 1, 20], dtype=torch.int32, device="cuda")
    want = moved(src, src, par.cpu(), 1, 3, lens.cpu())
    torch.cuda.synchronize()
    got = reorder_states(src, par, row_dim=1, length_dim=3, lengths=lens, stream=torch.cuda.Stream())
    torch.cuda.synchronize()
    assert torch.equal(got.cpu(), want.cpu())


def test_reorder_strided_views(hip):
    """A slice of a larger cache, rows not next to each other."""
    g = torch.Generator(device="cuda").manual_seed(2)
    cache = torch.randn(2, 8, 3, 50, 16, generator=g, device="cuda")
    view = cache[:, :6, 1:, :, :]
    par = torch.tensor([[1, 0, 2], [2, 2, 0]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([50, 13], dtype=torch.int32, device="cuda")
    want = cache.clone()
    want[:, :6, 1:] = moved(view, view, par.cpu(), 1, 3, lens.cpu())
    reorder_states(view, par, row_dim=1, length_dim=3, lengths=lens)
    torch.cuda.synchronize()
    assert torch.equal(cache, want)


def test_reorder_past_32_bits(hip):
    """Rows whose offsets pass 4 GiB."""
    rows, per = 6, 1 << 30
    state = torch.zeros(rows, per, dtype=torch.uint8, device="cuda")
    for r in range(rows):
        state[r, -1000:] = r + 1
        state[r, :1000] = 100 + r
    par = torch.tensor([[5, 5, 1, 0, 4, 2]], dtype=torch.int32, device="cuda")
    reorder_states(state, par)
    torch.cuda.synchronize()
    assert state[:, -1].tolist() == [6, 6, 2, 1, 5, 3] and state[:, 999].tolist() == [105, 105, 101, 100, 104, 102]
    assert state[:, 5000].tolist() == [0] * 6


def test_refusals(hip):
    bs = BeamSearch(2, 3, 100, 6)
    x, c = torch.zeros(6, 100, device="cuda"), torch.zeros(6, device="cuda")
    for bad in (lambda: bs.select(x[:5], c), lambda: bs.select(x[:, :99], c), lambda: bs.select(x.double(), c),
                lambda: bs.select(x, c[:5]), lambda: bs.select(x, c.double()), lambda: bs.select(x, c.cpu()),
                lambda: bs.select(x, c, finished=torch.zeros(6, dtype=torch.uint8, device="cuda")),
                lambda: bs.select(x, c, eos_id=100), lambda: bs.select(torch.zeros(9, 100, device="cuda"), c),
                lambda: bs.select(x, c, mask_words=torch.zeros(6, 3, dtype=torch.int32, device="cuda")),
                lambda: bs.select(torch.zeros(6, 200, device="cuda")[:, ::2], c)):
        with pytest.raises(ValueError):
            bad()
    for args in ((2, 33, 100, 6), (2, 3, 100, 65), (40000, 3, 100, 6), (2, 3, (1 << 23) + 1, 6)):
        with pytest.raises(_lib.HiRocmError):
            BeamSearch(*args)
    par = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    s = torch.zeros(6, 4, 8, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (lambda: reorder_states(s, par.long()), lambda: reorder_states(s[:5], par),
                lambda: reorder_states(s, par, dst=s.double()), lambda: reorder_states(s, par, length_dim=1),
                lambda: reorder_states(s, par, length_dim=0, lengths=lens),
                lambda: reorder_states(s.transpose(1, 2), par, length_dim=1, lengths=lens),
                lambda: reorder_states(s, par.cpu()), lambda: reorder_states(s.cpu(), par.cpu()),
                lambda: reorder_states(s[:, :0], par)):
        with pytest.raises(ValueError):
            bad()
    flat = torch.zeros(100, device="cuda")
    with pytest.raises(_lib.HiRocmError):  # rows that share bytes
        reorder_states(flat.as_strided((6, 8), (4, 1)), par)
    with pytest.raises(_lib.HiRocmError):  # dst overlaps src
        reorder_states(flat[:48].view(6, 8), par, dst=flat[8:56].view(6, 8))


def test_scores_in_place(hip):
    """With n_out = beams a step's scores and flags may replace the last one's."""
    B, K, V = 9, 4, 5000
    g = torch.Generator(device="cuda").manual_seed(5)
    bs = BeamSearch(B, K, V)
    x = torch.randn(B * K, V, generator=g, device="cuda").mul_(2.5)
    c = -torch.rand(B * K, generator=g, device="cuda")
    f = (torch.rand(B * K, generator=g, device="cuda") < 0.4).to(torch.uint8)
    want = bs.select(x, c.clone(), finished=f.clone(), eos_id=3)
    out = bs.outputs(B)
    out["scores"].copy_(c.view(B, K))
    out["finished"].copy_(f.view(B, K))
    got = bs.select(x, out["scores"], finished=out["finished"], eos_id=3, out=out)
    assert all(torch.equal(got[k], want[k]) for k in want)
    two = BeamSearch(B, K, V, 2 * K)
    with pytest.raises(ValueError):
        o = two.outputs(B)
        o["scores"] = c.view(-1)[:1].expand(1)  # (not even the right size)
        two.select(x, c, out=o)
    o = two.outputs(B)
    both = torch.empty(B * 2 * K, device="cuda")
    both[:B * K] = c
    o["scores"] = both
    with pytest.raises(ValueError, match="outputs over inputs"):
        two.select(x, both[:B * K], out=o)


def definition_on_gpu(x, c, mask, K, n):
    """`definition` without finished beams, rows all at once."""
    x = x.double().masked_fill(x.isnan(), -torch.inf)
    if mask is not None:
        x = x.masked_fill(~mask, -torch.inf)
    m = x.amax(1, keepdim=True)
    lse = m + (x - m).exp().sum(1, keepdim=True).log()
    top, ids = torch.sort(x, dim=1, descending=True, stable=True)
    top, ids = top[:, :n], ids[:, :n]
    score = torch.as_tensor(c, dtype=torch.float32).double().cuda()[:, None] + (top - lse)
    ok = torch.isfinite(score)
    big = lambda t: t[ok.expand_as(t)].abs().max().item()
    tol = EPS * (4 * big(lse.expand_as(score)) + 2 * big(top - lse) + 2 * big(score)) + SUM_EPS
    out = []
    for s, l, i, k in zip(*(t.view(-1, K, n).cpu().tolist() for t in (score, top, ids, ok))):
        cand = [(s[b][j], b, l[b][j], i[b][j]) for b in range(K) for j in range(n) if k[b][j]]
        out.append(sorted(cand, key=lambda t: (-t[0], t[1], -t[2], t[3])))
    return out, tol


def _streamed(kind, rows, V, dtype):
    """Rows for the kernel that streams a row through four waves."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(rows, V, generator=g, device="cuda").mul_(2.5)
    if kind == "few values":  # ties all over, also among the best
        x = (x * 2).round() / 2
    if kind == "odd":
        up = torch.arange(V, device="cuda", dtype=torch.float32)
        x[0] = up * 1e-3  # every tile holds better ones than those before it
        x[1] = -up * 1e-3
        x[2] = 1.0
        x[3, : V - 3] = -torch.inf
        x[4, ::3] = torch.nan
        x[8] = torch.where(up % 1000 == 999, 8.0, 0.0)
        x[9, V - 200:] = 50.0
    if kind == "extreme":  # (scores of these sizes leave only the order within a beam to check)
        x[5, :] = -3.0e38
        x[5, V // 2] = -2.9e38
        x[6, 7] = 3.0e38
        x[7] = (torch.arange(V, device="cuda") % 5) - 1e4
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind,K,V,n", [("plain", 8, 40000, 16), ("few values", 4, 40003, 8), ("few values", 8, 40000, 64),
                                        ("odd", 2, 40000, 16), ("odd", 2, 33333, 64), ("extreme", 2, 33333, 16), ("plain", 32, 25001, 64)])
def test_streamed_rows(hip, dtype, kind, K, V, n):
    rows = 1024
    x = _streamed(kind, rows, V, dtype)
    c = -np.random.default_rng(n).random(rows).astype(np.float32)
    res = run(x, c, K, n)
    want, tol = definition_on_gpu(x, c, None, K, n)
    check(res, want, tol, K, n, None, None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("share", [0.3, 0.001])
def test_streamed_masks(hip, dtype, share):
    rows, K, V, n = 2048, 4, 40000, 16
    x = _streamed("few values", rows, V, dtype)
    mask = torch.rand(rows, V, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < share
    mask[5] = False
    c = -np.random.default_rng(3).random(rows).astype(np.float32)
    res = run(x, c, K, n, mask=mask)
    want, tol = definition_on_gpu(x, c, mask, K, n)
    check(res, want, tol, K, n, None, None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,n", [(1, 32, 9000, 64), (2, 16, 8192 + 384, 64), (1, 32, 50257, 64), (3, 1, 4096 + 1105, 64),
                                     (2, 7, 37000, 56), (1, 32, 151936, 64), (5, 3, 8192 + 3, 40)])
def test_many_candidates(hip, dtype, B, K, V, n):
    """Parts that end early, and as many candidates as a request may keep."""
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(B * K, V, generator=g, device="cuda").mul_(2.5).to(dtype)
    for spread in (0.5, 40.0):
        c = (-np.random.default_rng(K).random(B * K) * spread).astype(np.float32)
        res = run(x, c, K, n)
        want, tol = definition_on_gpu(x, c, None, K, n)
        check(res, want, tol, K, n, None, None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [2048, 4999, 40000])
@pytest.mark.parametrize("n", [1, 8, 64])
def test_signalling_nan(hip, dtype, V, n):
    """NaN logits of either kind count as masked, wherever they lie beside a
    row's largest logits: at each of eight neighbours of the largest one, in
    every other place, in all of a part but one place."""
    rng = np.random.default_rng(V + n)
    x = torch.from_numpy(rng.standard_normal((56 + 8, V)).astype(np.float32) * 2.5).cuda().to(dtype)
    nan = torch.zeros(x.shape, dtype=torch.bool, device="cuda")
    for r in range(56):
        best, other = r // 7, r % 7
        other += other >= best
        at = int(rng.integers(0, V // 8)) * 8
        x[r, at + best] = 20.0
        nan[r, at + other] = True
    for r in range(56, 64):
        nan[r, r % 2::2] = True                    # every other place
        if r >= 60:
            nan[r] = True                          # all, but one place of each 1,000
            nan[r, r % 8::1000] = False
    bits, word = (torch.int32, 0x7f800001) if dtype is torch.float32 else (torch.int16, 0x7f81)
    x.view(bits)[nan] = word
    c = -rng.random(64).astype(np.float32)
    with np.errstate(invalid="ignore"):  # (numpy's cast of a signalling NaN)
        agree(x, c, 1, n)
    if V == 40000:  # rows enough for the kernel that streams them
        many = x.repeat(16, 1)
        res = run(many, np.tile(c, 16), 1, n)
        want, tol = definition_on_gpu(many, np.tile(c, 16), None, 1, n)
        check(res, want, tol, 1, n, None, None)


def test_equal_logits_of_waves_apart(hip):
    """The lower token among equal logits, where one wave of a part is far
    behind the others.  The first wave's tiles (1,024 logits, every fourth) rise
    in steps that fill its list; the others have little to list, and 16 lanes of
    each reach 2 at their eighth tile, before the first wave gets to its fifth:
    there 16 lanes reach 2, in its sixth 48 more.  Those 64 come before the
    others' 48."""
    rows, V, n, tile = 1024, 40000, 64, 1024
    row = torch.full((V,), 0.5)
    at = lambda step, wave: (step * 4 + wave) * tile
    for wave in range(4):
        row[at(0, wave):at(0, wave) + tile] = 1.0
    row[at(1, 0):at(1, 0) + tile] = 1.25
    row[at(2, 0):at(2, 0) + tile] = 1.5
    row[at(3, 0):at(3, 0) + tile * 3 // 4] = 1.75
    first = [at(4, 0) + 4 * lane for lane in range(16)] + [at(5, 0) + 4 * lane for lane in range(48)]
    later = [at(7, wave) + 4 * lane for wave in (1, 2, 3) for lane in range(16)]
    row[first + later] = 2.0
    x = row.cuda().repeat(rows, 1)
    res = run(x, np.zeros(rows, np.float32), 1, n)
    assert (res["tokens"].cpu() == torch.tensor(first, dtype=torch.int32)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("requests,V", [(2, 9001), (170, 40000)])
def test_scores_beside_special_rows(hip, dtype, requests, V):
    """Beams with NaN, infinite, equal and single logits among ordinary ones,
    and none whose size would widen the scores' bound: by both kernels."""
    K, n = 6, 12
    rng = np.random.default_rng(V)
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(requests * K, V, generator=g, device="cuda").mul_(2.5).to(dtype)
    x[0, 10:20] = torch.nan
    x[0, 0] = torch.nan
    x[1] = torch.nan                  # no candidate
    x[2, 5] = torch.inf               # none either
    x[3] = -torch.inf
    x[3, 77] = 1.0                    # one candidate of probability 1
    x[4, ::2] = -torch.inf
    x[6] = 0.0
    x[6, 1::2] = -0.0                 # equal to 0: the lower token first
    x[7, V - 1] = 30.0                # probability 1 but for rounding
    x[8, : V - 3] = -torch.inf
    c = -rng.random(requests * K).astype(np.float32) * 8
    c[9], c[10], c[11] = -np.inf, np.nan, np.inf
    for beams in (K, 1):  # (as requests of their own every row's scores are seen)
        res = run(x, c, beams, n)
        want, tol = definition_on_gpu(x, c, None, beams, n)
        assert tol < 3e-5
        check(res, want, tol, beams, n, None, None)

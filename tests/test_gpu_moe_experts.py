"""The expert layer against the definitions in 64 bits.

A product of k terms in f32 is off by at most k eps times the sum of their
magnitudes; silu(g) u by |u| 1.1 dg + |silu(g)| du and a few eps of itself;
a bf16 result by half a unit of its last place more."""
import numpy as np
import pytest
import torch

from hi_amd import _lib
from hi_amd.moe import MoeExperts, RowGroups, combine, group_rows, grouped_product

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def routes(tokens, top_k, experts, seed, kind="spread"):
    g = gen(seed)
    if kind == "one":  # every pair to one expert
        return torch.full((tokens, top_k), experts - 1, dtype=torch.int32, device="cuda")
    if kind == "few":
        return torch.randint(0, min(2, experts), (tokens, top_k), generator=g, device="cuda").int()
    ids = torch.randint(0, experts, (tokens, top_k), generator=g, device="cuda").int()
    if kind == "strays":  # ids that name no expert
        ids[torch.rand(tokens, top_k, generator=g, device="cuda") < 0.3] = -1
        ids[0, 0] = experts
    return ids


def definition(ids, experts):
    v = ids.cpu().numpy().astype(np.int64).ravel()
    v = np.where((v < 0) | (v >= experts), experts, v)
    order = np.argsort(v, kind="stable")
    slots = np.empty_like(order)
    slots[order] = np.arange(order.size)
    offsets = np.searchsorted(v[order], np.arange(experts + 1))
    return order, slots, offsets


@pytest.mark.parametrize("kind", ["spread", "one", "few", "strays"])
@pytest.mark.parametrize("tokens,top_k,experts", [(1, 1, 1), (1, 8, 256), (5, 3, 7), (64, 2, 64), (300, 4, 60),
                                                  (4096, 1, 3), (1025, 4, 2048), (9001, 8, 128)])
def test_grouping(hip, tokens, top_k, experts, kind):
    ids = routes(tokens, top_k, experts, tokens, kind)
    got = group_rows(ids, experts)
    torch.cuda.synchronize()
    order, slots, offsets = definition(ids, experts)
    assert np.array_equal(got.order.cpu().numpy(), order)
    assert np.array_equal(got.slots.cpu().numpy(), slots)
    assert np.array_equal(got.offsets.cpu().numpy(), offsets)


def product(x, w, order, offsets, top_k, gather, swiglu):
    """The products in the groups' order and their bound."""
    places, k = order.size, w.shape[2]
    wide = w.shape[1] // 2 if swiglu else w.shape[1]
    y = torch.zeros(places, wide, dtype=torch.float64)
    tol = torch.zeros_like(y)
    xx = x.double().cpu()
    for e in range(w.shape[0]):
        a, b = int(offsets[e]), int(offsets[e + 1])
        if a == b:
            continue
        rows = torch.from_numpy(order[a:b] // top_k) if gather else torch.arange(a, b)
        we = w[e].double().cpu()
        r = xx[rows] @ we.t()
        d = (k + 8) * EPS * (xx[rows].abs() @ we.abs().t())
        if swiglu:
            g, u, dg, du = r[:, :wide], r[:, wide:], d[:, :wide], d[:, wide:]
            silu = g / (1 + torch.exp(-g))
            r, d = silu * u, u.abs() * 1.1 * dg + silu.abs() * du + 8 * EPS * (silu * u).abs()
        y[a:b], tol[a:b] = r, d
    return y, tol


def agree(got, y, tol, end):
    """Within the bound; a bf16 result is the rounding of a value within it."""
    got, y, tol = got[:end].cpu(), y[:end], tol[:end]
    if got.dtype == torch.bfloat16:
        assert ((got >= (y - tol).float().bfloat16()) & (got <= (y + tol).float().bfloat16())).all()
        return
    d = (got.double() - y).abs()
    assert (d <= tol).all(), (d - tol).max()


def half_unit(y):
    """Half a unit of bf16's last place (8 significant bits)."""
    return torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -126))) - 8)


SIZES = [(1, 1, 1, 1, 8), (1, 2, 4, 16, 32), (3, 2, 5, 18, 40), (8, 8, 64, 96, 256), (33, 4, 6, 130, 72),
         (200, 4, 9, 72, 104), (257, 2, 3, 520, 64), (600, 1, 2, 258, 200), (1200, 2, 5, 384, 512),
         (3000, 2, 4, 256, 128)]


@pytest.mark.parametrize("kind", ["spread", "one", "strays"])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("tokens,top_k,experts,cols,k", SIZES)
def test_products(hip, tokens, top_k, experts, cols, k, swiglu, kind):
    if swiglu and cols % 2:
        cols += 1
    ids = routes(tokens, top_k, experts, tokens + k, kind)
    g = gen(cols)
    x = torch.randn(tokens, k, generator=g, device="cuda").bfloat16()
    w = (torch.randn(experts, cols, k, generator=g, device="cuda") * k ** -0.5).bfloat16()
    groups = group_rows(ids, experts)
    order, _, offsets = definition(ids, experts)
    y, tol = product(x, w, order, offsets, top_k, True, swiglu)
    end = int(offsets[-1])
    wide = cols // 2 if swiglu else cols
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((tokens * top_k, wide + 3), 77.0, dtype=dtype, device="cuda")
        grouped_product(x, w, groups, swiglu=swiglu, out=out[:, :wide])
        torch.cuda.synchronize()
        agree(out[:, :wide], y, tol, end)
        assert (out[:, wide:] == 77.0).all() and (out[end:] == 77.0).all()  # nothing else is written


@pytest.mark.parametrize("tokens,top_k,experts,cols,k", [(4, 2, 8, 48, 64), (300, 2, 3, 200, 96), (900, 2, 4, 256, 128)])
def test_rows_in_group_order_and_strided(hip, tokens, top_k, experts, cols, k):
    ids = routes(tokens, top_k, experts, 1)
    groups = group_rows(ids, experts)
    order, _, offsets = definition(ids, experts)
    big = torch.full((tokens * top_k, k + 24), float("nan"), device="cuda").bfloat16()
    x = big[:, 8:8 + k]
    x.copy_(torch.randn(tokens * top_k, k, generator=gen(3), device="cuda"))
    w = (torch.randn(experts, cols, k, generator=gen(4), device="cuda") * k ** -0.5).bfloat16()
    y, tol = product(x, w, order, offsets, top_k, False, False)
    agree(grouped_product(x, w, groups, gather=False, dtype=torch.float32), y, tol, tokens * top_k)


def test_values_that_do_not_mix(hip):
    """inf and NaN in one row of x and in one expert reach only their own
    places; weights past 32-bit offsets."""
    tokens, top_k, experts, cols, k = 40, 2, 5, 64, 96
    ids = routes(tokens, top_k, experts, 7)
    groups = group_rows(ids, experts)
    x = torch.randn(tokens, k, generator=gen(1), device="cuda").bfloat16()
    w = torch.randn(experts, cols, k, generator=gen(2), device="cuda").bfloat16()
    clean = grouped_product(x, w, groups, dtype=torch.float32)
    x2, w2 = x.clone(), w.clone()
    x2[3, 5], w2[2] = float("inf"), float("nan")
    got = grouped_product(x2, w2, groups, dtype=torch.float32)
    pairs = groups.order.long()
    own = (ids.view(-1)[pairs] != 2) & (pairs // top_k != 3)
    assert torch.equal(clean[own], got[own]) and own.sum() > 10
    assert got[ids.view(-1)[pairs] == 2].isnan().all()


def test_weights_past_32_bits(hip):
    """Experts whose weights start beyond 2^32 elements."""
    experts, cols, k = 9, 16384, 32768
    w = torch.zeros(experts, cols, k, dtype=torch.bfloat16, device="cuda")
    w[8, :, 5] = 2.0
    w[8, 16383, 32767] = 1.0
    w[0, :, 5] = 1.0
    x = torch.ones(2, k, device="cuda").bfloat16()
    groups = group_rows(torch.tensor([[8], [0]], dtype=torch.int32, device="cuda"), experts)
    y = grouped_product(x, w, groups, dtype=torch.float32)
    assert (y[0] == 1.0).all() and (y[1, :-1] == 2.0).all() and float(y[1, -1]) == 3.0


@pytest.mark.parametrize("ydtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("odtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,top_k,cols", [(1, 1, 1), (7, 3, 33), (130, 8, 264), (70000, 1, 3), (40, 2, 1024)])
def test_combination(hip, tokens, top_k, cols, ydtype, odtype):
    ids = routes(tokens, top_k, 6, 5, "strays" if tokens > 1 else "spread")
    groups = group_rows(ids, 6)
    _, slots, offsets = definition(ids, 6)
    y = torch.randn(tokens * top_k, cols, generator=gen(6), device="cuda").to(ydtype)
    y[int(offsets[-1]):] = float("nan")  # no product there
    wts = torch.rand(tokens, top_k, generator=gen(7), device="cuda")
    got = combine(y, groups, wts, dtype=odtype)
    yy = y.double().cpu().nan_to_num(0.0)[torch.from_numpy(slots)].view(tokens, top_k, cols)
    t = yy * wts.double().cpu()[:, :, None]
    agree(got, t.sum(1), (top_k + 2) * EPS * t.abs().sum(1), tokens)


@pytest.mark.parametrize("tokens", [1, 5, 200])
def test_layer(hip, tokens):
    """The layer as a whole: bf16 activations between the products add half a
    unit of their last place each, which the second product carries as any
    other error of its inputs."""
    E, H, I, k = 12, 104, 56, 3
    g = gen(tokens)
    up = (torch.randn(E, 2 * I, H, generator=g, device="cuda") * H ** -0.5).bfloat16()
    down = (torch.randn(E, H, I, generator=g, device="cuda") * I ** -0.5).bfloat16()
    layer = MoeExperts(up, down, max_tokens=200, top_k=k)
    x = torch.randn(tokens, H, generator=g, device="cuda").bfloat16()
    ids = routes(tokens, k, E, tokens)
    wts = torch.softmax(torch.randn(tokens, k, generator=g, device="cuda"), 1)
    order, slots, offsets = definition(ids, E)
    h, dh = product(x, up, order, offsets, k, True, True)
    dh = dh + half_unit(h.abs() + dh)
    y, dy = product(h, down, order, offsets, k, False, False)
    carried, _ = product(dh, down.abs(), order, offsets, k, False, False)
    back = torch.from_numpy(slots)
    w = wts.double().cpu()[:, :, None]
    want = (y[back].view(tokens, k, H) * w).sum(1)
    tol = ((dy + carried)[back].view(tokens, k, H) * w).sum(1) * 1.001
    got = layer(x, ids, wts)
    agree(got, want, tol, tokens)
    assert torch.equal(layer(x, ids, wts), got)  # the same bits again


def test_streams_and_graph(hip):
    E, H, I, k, T = 8, 64, 32, 2, 24
    g = gen(1)
    layer = MoeExperts(torch.randn(E, 2 * I, H, generator=g, device="cuda").bfloat16(),
                       torch.randn(E, H, I, generator=g, device="cuda").bfloat16(), T, k)
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    ids, wts = routes(T, k, E, 2), torch.rand(T, k, generator=g, device="cuda")
    out = torch.empty_like(x)
    layer(x, ids, wts, out=out)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        layer(x, ids, wts, out=out)
    for i in range(4):
        x.copy_(torch.randn(T, H, generator=g, device="cuda"))
        ids.copy_(routes(T, k, E, 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, layer(x, ids, wts))


def test_refusals(hip):
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    w = torch.zeros(3, 16, 32, device="cuda").bfloat16()
    x = torch.zeros(4, 32, device="cuda").bfloat16()
    groups = group_rows(ids, 3)
    for bad in (lambda: group_rows(ids.long(), 3), lambda: group_rows(ids[0], 3), lambda: group_rows(ids[:0], 3),
                lambda: group_rows(ids.cpu(), 3), lambda: group_rows(ids, 3, out=RowGroups(4, 2, 4)),
                lambda: grouped_product(x[:3], w, groups), lambda: grouped_product(x.float(), w, groups),
                lambda: grouped_product(x, w[:2], groups), lambda: grouped_product(x, w.float(), groups),
                lambda: grouped_product(x, w, groups, gather=False), lambda: grouped_product(x.cpu(), w, groups),
                lambda: grouped_product(x, w[:, :15].contiguous(), groups, swiglu=True),
                lambda: grouped_product(x, w, groups, out=torch.zeros(8, 15, device="cuda")),
                lambda: combine(torch.zeros(7, 5, device="cuda"), groups, torch.zeros(4, 2, device="cuda")),
                lambda: combine(torch.zeros(8, 5, device="cuda"), groups, torch.zeros(4, 3, device="cuda")),
                lambda: MoeExperts(w, w, 4, 2)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.HiRocmError):
        group_rows(ids, 2049)
    with pytest.raises(_lib.HiRocmError):  # k no multiple of 8
        grouped_product(torch.zeros(4, 12, device="cuda").bfloat16(),
                        torch.zeros(3, 16, 12, device="cuda").bfloat16(), groups)
    wide = torch.zeros(4, 64, device="cuda").bfloat16()
    with pytest.raises(_lib.HiRocmError):  # rows that do not start on 16 bytes
        grouped_product(wide[:, 4:36], w, groups)


@pytest.mark.parametrize("kind", ["spread", "one", "strays"])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("tokens,top_k,experts,cols,k", [(1200, 1, 40, 1030, 72), (2000, 2, 24, 1536, 136),
                                                         (4800, 1, 16, 2048, 104), (2500, 4, 12, 1800, 64)])
def test_products_of_many_workgroups(hip, tokens, top_k, experts, cols, k, swiglu, kind):
    """Tiles of 128 and of 256 places with more workgroups than half the card's
    CUs, into rows that can and that cannot be written 16 bytes at a time."""
    ids = routes(tokens, top_k, experts, tokens + k, kind)
    g = gen(cols)
    x = torch.randn(tokens, k, generator=g, device="cuda").bfloat16()
    w = (torch.randn(experts, cols, k, generator=g, device="cuda") * k ** -0.5).bfloat16()
    groups = group_rows(ids, experts)
    order, _, offsets = definition(ids, experts)
    y, tol = product(x, w, order, offsets, top_k, True, swiglu)
    end = int(offsets[-1])
    wide = cols // 2 if swiglu else cols
    for dtype in (torch.float32, torch.bfloat16):
        for pad in (0, 3):
            out = torch.full((tokens * top_k, wide + pad), 77.0, dtype=dtype, device="cuda")
            grouped_product(x, w, groups, swiglu=swiglu, out=out[:, :wide])
            torch.cuda.synchronize()
            agree(out[:, :wide], y, tol, end)
            assert (out[:, wide:] == 77.0).all() and (out[end:] == 77.0).all()


@pytest.mark.parametrize("tokens,experts,inter", [(40, 5, 40), (60, 5, 40), (200, 5, 40), (2400, 40, 520), (4000, 4, 3820)])
def test_gates_of_any_size(hip, tokens, experts, inter):
    """silu(gate) up over gates from -400 to 400, every 0.1 from -130 to 130, by
    each product kernel: 8 and 12 places an expert, 40, 60 with more workgroups
    than half the card's CUs, and 1,000.

    Gates are multiples of 2^-8 below 512, given as the sum of two bf16 weights,
    and ups small whole numbers, so both sums are exact.  What is left: the
    exponential (2 eps), its correction (1), 1 + e (1), the reciprocal (2), two
    products (2) and the correction's own terms (2); a reciprocal below the
    smallest normal number may be taken as 0, which is off by |g u| 2^-126."""
    ids = (torch.arange(tokens, device="cuda", dtype=torch.int32) % experts).view(-1, 1)
    groups = group_rows(ids, experts)
    g = torch.cat((torch.linspace(-130.0, 130.0, 2601), torch.tensor([-400.0, -150.0, -88.7228, 88.7229, 150.0, 400.0])))
    g = (g.double() * 256).round().cuda() / 256
    x = torch.zeros(tokens, 64, device="cuda").bfloat16()
    x[:, :2] = 1.0
    x[:, 2] = torch.arange(1, tokens + 1, device="cuda") % 7 - 3.0
    w = torch.zeros(experts, 2 * inter, 64, device="cuda").bfloat16()
    w[:, inter:, 2] = 1.0
    places = groups.order.long()
    for first in range(0, g.numel(), experts * inter):
        gate = g[(first + torch.arange(experts * inter, device="cuda")) % g.numel()].view(experts, inter)
        w[:, :inter, 0] = gate.float().bfloat16()
        w[:, :inter, 1] = (gate - w[:, :inter, 0].double()).float().bfloat16()
        got = grouped_product(x, w, groups, swiglu=True, dtype=torch.float32).double()
        up = x[places, 2].double()[:, None]
        gate = gate[ids.view(-1).long()[places]]
        want = gate / (1.0 + torch.exp(-gate)) * up
        tol = 10 * EPS * want.abs() + (gate * up).abs() * 2.0 ** -126
        bad = ~((got - want).abs() <= tol)
        assert not bad.any(), (first, gate[bad][:5].tolist(), got[bad][:5].tolist(), want[bad][:5].tolist())


@pytest.mark.parametrize("kind", ["spread", "one"])
@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("tokens,top_k,experts,cols,k", [(16, 4, 16, 100, 704), (3, 2, 6, 70, 2056), (75, 4, 20, 136, 520),
                                                         (64, 2, 8, 130, 1032), (150, 2, 6, 200, 1000),
                                                         (1200, 1, 40, 1030, 520), (2000, 2, 24, 1536, 520)])
def test_products_over_many_steps(hip, tokens, top_k, experts, cols, k, swiglu, kind):
    """Each product kernel with k of many more steps than it has buffers: 4, 1,
    15 and 16 places an expert, 50, 30 and 166 with more workgroups."""
    ids = routes(tokens, top_k, experts, tokens + k, kind)
    g = gen(cols)
    x = torch.randn(tokens, k, generator=g, device="cuda").bfloat16()
    w = (torch.randn(experts, cols, k, generator=g, device="cuda") * k ** -0.5).bfloat16()
    groups = group_rows(ids, experts)
    order, _, offsets = definition(ids, experts)
    y, tol = product(x, w, order, offsets, top_k, True, swiglu)
    for dtype in (torch.float32, torch.bfloat16):
        agree(grouped_product(x, w, groups, swiglu=swiglu, dtype=dtype), y, tol, tokens * top_k)


@pytest.mark.parametrize("tokens,k,E,H,I", [(70, 4, 20, 520, 264), (300, 4, 10, 1032, 136), (1000, 4, 24, 1536, 768)])
def test_larger_layers(hip, tokens, k, E, H, I):
    """As test_layer, by the kernels for more places an expert."""
    g = gen(tokens)
    up = (torch.randn(E, 2 * I, H, generator=g, device="cuda") * H ** -0.5).bfloat16()
    down = (torch.randn(E, H, I, generator=g, device="cuda") * I ** -0.5).bfloat16()
    x = torch.randn(tokens, H, generator=g, device="cuda").bfloat16()
    ids = routes(tokens, k, E, tokens, "strays")
    wts = torch.softmax(torch.randn(tokens, k, generator=g, device="cuda"), 1)
    order, slots, offsets = definition(ids, E)
    h, dh = product(x, up, order, offsets, k, True, True)
    dh = dh + half_unit(h.abs() + dh)
    y, dy = product(h, down, order, offsets, k, False, False)
    carried, _ = product(dh, down.abs(), order, offsets, k, False, False)
    back = torch.from_numpy(slots)
    w = wts.double().cpu()[:, :, None]
    want = (y[back].view(tokens, k, H) * w).sum(1)
    tol = ((dy + carried)[back].view(tokens, k, H) * w).sum(1) * 1.001
    out = torch.empty(tokens, H, device="cuda")
    layer = MoeExperts(up, down, max_tokens=tokens + 5, top_k=k)
    agree(layer(x, ids, wts, out=out), want, tol, tokens)
    agree(layer(x, ids, wts), want, tol, tokens)

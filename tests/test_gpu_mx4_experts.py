"""The expert layer with 4-bit products against its definition in 64 bits.

The first product is held to the bound of tests/test_gpu_mx4.py.  Behind silu and
the product with up, relative errors of some 2^-20 can move an activation over a
border between two codes, a step of its block: the layer is compared with the
layer that goes on from the kernel's own rounded activations, and those
activations with the exact ones, code by code, but next to borders."""
import pytest
import torch

from hi_amd import _lib, mx4
from hi_amd.beam import _CODES
from hi_amd.moe import RowGroups, combine, group_rows
from hi_amd.mx4 import Mx4Experts
from oracle import mx4_oracle as O

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -23


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def weights(E, n, k, seed):
    g = gen(seed)
    w = torch.randn(E * n, k, generator=g, device="cuda") * k ** -0.5
    codes, scales = mx4.quantize_mx4(w)
    return codes.view(E, n, k // 2), scales.view(E, n, k // 32)


def route(T, E, K, seed, none=0.0):
    g = gen(seed)
    ids = torch.rand(T, E, generator=g, device="cuda").topk(min(K, E), 1).indices.int()
    if ids.size(1) < K:
        ids = torch.cat((ids, ids.new_full((T, K - ids.size(1)), -1)), 1)
    ids = torch.where(torch.rand(T, K, generator=g, device="cuda") < none, torch.full_like(ids, E), ids).contiguous()
    w = torch.rand(T, K, generator=g, device="cuda")
    return ids, w / w.sum(1, keepdim=True)


def product(x, packed, groups, cols, k, swiglu=False, gather=True, dtype=torch.float32, out=None, work=None):
    """hi_rocm_mx4_grouped_product on a bf16 x (or Mx4Rows)."""
    lib, wide = _lib.load(), cols // 2 if swiglu else cols
    if out is None:
        out = torch.full((groups.places, wide), 55.0, dtype=dtype, device="cuda")
    to_rows = isinstance(out, mx4.Mx4Rows)
    if isinstance(x, mx4.Mx4Rows):
        at, code, rows, stride = x.memory, _lib.DTYPE_MX4, x.rows, 0
    else:
        at, code, rows, stride = x, _lib.DTYPE_BF16, x.size(0), x.stride(0)
        work = torch.empty(mx4._size(lib.hi_rocm_mx4_rows_bytes, rows, k), dtype=torch.uint8, device="cuda")
    memory = out.memory if to_rows else out
    _lib.check(lib.hi_rocm_mx4_grouped_product(
        at.data_ptr(), code, rows, stride, groups.order.data_ptr() if gather else 0, groups.top_k,
        groups.offsets.data_ptr(), groups.places, groups.experts, packed.data_ptr(), packed.numel(), cols, k, int(swiglu),
        memory.data_ptr(), _lib.DTYPE_MX4 if to_rows else _CODES[out.dtype], 0 if to_rows else out.stride(0),
        memory.numel() if to_rows else 0, 0 if work is None else work.data_ptr(), 0 if work is None else work.numel(),
        torch.cuda.current_stream().cuda_stream))
    return out


def values_of(rows):
    """The values (float64) and scale bytes of Mx4Rows."""
    k, n = rows.k, rows.rows
    quads, begin = -(-k // 512), n * (k // 2)
    codes = rows.memory[:begin].view(n, k // 2)
    s = rows.memory[begin:begin + n * quads * 16].view(n, quads, 4, 4)  # [g][j]: block 4 j + g
    s = s.transpose(2, 3).reshape(n, quads * 16)[:, :k // 32].contiguous()
    return O.values(codes.contiguous(), s), s.cpu()


def in_places(groups, ids, E):
    """Each place's token and expert (-1: none), on the CPU."""
    order = groups.order.cpu().long()
    return order // groups.top_k, torch.where((ids.view(-1).cpu()[order] >= 0) & (ids.view(-1).cpu()[order] < E),
                                              ids.view(-1).cpu()[order].long(), torch.tensor(-1))


SIZES = [(1, 1, 1, 32, 32), (1, 4, 2, 64, 32), (5, 8, 2, 96, 64), (16, 3, 3, 160, 96), (17, 60, 4, 320, 160),
         (64, 7, 2, 544, 96), (200, 16, 4, 512, 224), (300, 4, 2, 1184, 352), (700, 8, 4, 256, 128)]


# Few experts with some places each: narrow tiles that share a long k out, larger tiles
NARROW = [(30, 8, 4, 2080, 1056), (26, 4, 2, 1568, 96), (50, 5, 3, 4640, 64), (90, 16, 2, 1440, 1536), (9, 1, 1, 3680, 544),
          (120, 8, 4, 1056, 2592), (460, 2, 2, 608, 1056), (135, 16, 2, 32, 1920), (280, 16, 3, 32, 1728)]


@pytest.mark.parametrize("T,E,K,H,I", SIZES + NARROW)
@pytest.mark.parametrize("none", [0.0, 0.3])
def test_products(hip, T, E, K, H, I, none):
    """Both products on their own: gathered bf16 rows, rows in the groups' order,
    f32 and bf16; places behind the groups stay as they were."""
    K = min(K, E)
    ids, _ = route(T, E, K, seed=T, none=none)
    up, ups = weights(E, 2 * I, H, seed=E)
    packed = mx4._pack("test", up, ups, E, None)
    x = torch.randn(T, H, generator=gen(3), device="cuda").bfloat16()
    groups = group_rows(ids, E)
    token, expert = in_places(groups, ids, E)
    xx = O.rounded(x)[token]
    w = O.values(up, ups)
    n = int(groups.offsets[E])
    y = torch.stack([w[e] @ r for e, r in zip(expert[:n], xx[:n])]) if n else torch.zeros(0, 2 * I, dtype=torch.float64)
    size = torch.stack([w[e].abs() @ r.abs() for e, r in zip(expert[:n], xx[:n])]) if n else y
    tol = (H // 32 + 8) * STEP * size
    got = product(x, packed, groups, 2 * I, H)
    assert ((got[:n].double().cpu() - y).abs() <= tol).all()
    assert (got[n:] == 55).all()
    b = product(x, packed, groups, 2 * I, H, dtype=torch.bfloat16)[:n].cpu()
    assert ((b >= (y - tol).float().bfloat16()) & (b <= (y + tol).float().bfloat16())).all()
    rows = mx4.mx4_rows(x.float()[token.cuda()])
    assert torch.equal(product(rows, packed, groups, 2 * I, H, gather=False)[:n], product(
        mx4.mx4_rows(x), packed, groups, 2 * I, H)[:n])
    # silu(gate) up: the gate's and up's errors, 8 steps of silu's own
    gate, u = y[:, :I], y[:, I:]
    h = torch.nn.functional.silu(gate) * u
    ht = 1.1 * tol[:, :I] * u.abs() + 1.1 * gate.abs() * tol[:, I:] + 1.1 * tol[:, :I] * tol[:, I:] + 8 * STEP * h.abs()
    act = product(x, packed, groups, 2 * I, H, swiglu=True)
    assert ((act[:n].double().cpu() - h).abs() <= ht).all()
    assert (act[n:] == 55).all()
    # and rounded: the rounding of the f32 activations
    out = mx4.Mx4Rows(groups.places, I)
    out.memory.fill_(0xA5)
    product(x, packed, groups, 2 * I, H, swiglu=True, out=out)
    v, s = values_of(out)
    codes, scales = O.quantize(act[:n])
    assert torch.equal(s[:n], scales)
    assert torch.equal(v[:n], O.values(O.pack_nibbles(codes), scales))
    assert (s[n:] == 0xA5).all()


@pytest.mark.parametrize("T,E,K,H,I", SIZES + NARROW)
@pytest.mark.parametrize("none", [0.0, 0.3])
def test_layer(hip, T, E, K, H, I, none):
    K = min(K, E)
    ids, wts = route(T, E, K, seed=T + 1, none=none)
    up, ups = weights(E, 2 * I, H, seed=E)
    down, downs = weights(E, H, I, seed=E + 1)
    x = torch.randn(T, H, generator=gen(4), device="cuda").bfloat16()
    layer = Mx4Experts(up, ups, down, downs, max_tokens=T + 3, top_k=K)
    out32 = layer(x, ids, wts, out=torch.empty(T, H, device="cuda"))
    got = layer(x, ids, wts).cpu()
    # from the kernel's own activations
    groups = group_rows(ids, E)
    h = mx4.Mx4Rows(groups.places, I)
    product(x, mx4._pack("test", up, ups, E, None), groups, 2 * I, H, swiglu=True, out=h)
    n = int(groups.offsets[E])
    v, _ = values_of(h)
    _, expert = in_places(groups, ids, E)
    w = O.values(down, downs)
    y, size = torch.zeros(groups.places, H, dtype=torch.float64), torch.zeros(groups.places, H, dtype=torch.float64)
    for i in range(n):
        y[i], size[i] = w[expert[i]] @ v[i], w[expert[i]].abs() @ v[i].abs()
    slots, ww = groups.slots.cpu().long(), wts.double().cpu()
    want = (y[slots].view(T, K, H) * ww[:, :, None]).sum(1)
    tol = ((I // 32 + 8 + K + 2) * STEP * size[slots].view(T, K, H) * ww[:, :, None]).sum(1)
    assert ((out32.double().cpu() - want).abs() <= tol).all()
    # bf16 terms are off by another half step each, 2^-8 of what is within their bound
    bound = tol + 1.01 * 2.0 ** -8 * (y[slots].abs().view(T, K, H) * ww[:, :, None]).sum(1) + 2.0 ** -7 * tol
    assert ((got >= (want - bound).float().bfloat16()) & (got <= (want + bound).float().bfloat16())).all()
    # the activations against the exact ones: a code a step away only next to a border
    token, _ = in_places(groups, ids, E)
    xx, wu = O.rounded(x)[token], O.values(up, ups)
    if n:
        g = torch.stack([wu[e] @ r for e, r in zip(expert[:n], xx[:n])])
        exact = torch.nn.functional.silu(g[:, :I]) * g[:, I:]
        assert (v[:n] != O.rounded(exact)).sum() <= 1 + n * I // 10000


@pytest.mark.parametrize("cols", [1, 50, 300, 1000])
@pytest.mark.parametrize("T,E,K,H", [(3, 5, 2, 96), (90, 3, 2, 384), (2, 1, 40, 160), (700, 6, 3, 896)])
def test_any_number_of_columns(hip, T, E, K, H, cols):
    """Columns that end inside tiles and blocks, more pairs of an expert than
    tokens; rows of the same places in any form."""
    g = gen(T)
    ids = torch.randint(0, E, (T, K), generator=g, device="cuda").int()
    w, s = weights(E, cols, H, seed=cols)
    packed = mx4._pack("test", w, s, E, None)
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    groups = group_rows(ids, E)
    token, expert = in_places(groups, ids, E)
    xx, ww = O.rounded(x)[token], O.values(w, s)
    y = torch.stack([ww[e] @ r for e, r in zip(expert, xx)])
    tol = (H // 32 + 8) * STEP * torch.stack([ww[e].abs() @ r.abs() for e, r in zip(expert, xx)])
    out = torch.full((T * K, cols + 5), 55.0, device="cuda")
    product(x, packed, groups, cols, H, out=out[:, :cols])
    assert ((out[:, :cols].double().cpu() - y).abs() <= tol).all() and (out[:, cols:] == 55).all()
    got = product(mx4.mx4_rows(x), packed, groups, cols, H)
    assert ((got.double().cpu() - y).abs() <= tol).all()


def test_prepared_together(hip):
    """Groups and rows from one launch are those of two."""
    lib = _lib.load()
    for T, E, K, H in ((1, 3, 1, 32), (20, 60, 4, 1440), (3000, 17, 6, 544)):
        ids, _ = route(T, E, K, seed=T, none=0.1)
        x = torch.randn(T, H + 32, generator=gen(T), device="cuda").bfloat16()[:, :H]
        want, rows = group_rows(ids, E), mx4.mx4_rows(x)
        got, out = RowGroups(T, K, E), mx4.Mx4Rows(T, H)
        for t in (got.order, got.slots, got.offsets):
            t.fill_(-7)
        _lib.check(lib.hi_rocm_mx4_moe_prepare(
            ids.data_ptr(), T, K, E, got.order.data_ptr(), got.slots.data_ptr(), got.offsets.data_ptr(), x.data_ptr(), H,
            x.stride(0), out.memory.data_ptr(), out.memory.numel(), torch.cuda.current_stream().cuda_stream))
        n = int(want.offsets[E])
        assert torch.equal(got.offsets, want.offsets) and torch.equal(got.order, want.order)
        assert torch.equal(got.slots, want.slots) and 0 <= n <= T * K
        for a, b in zip(values_of(out), values_of(rows)):
            assert torch.equal(a, b)


def test_fused_rows_and_workspace_agree(hip):
    """Rows rounded as they are read (up to 16) and beforehand: the same values,
    so sums that differ by their order alone."""
    E, H, I, K = 4, 512, 64, 2
    up, ups = weights(E, 2 * I, H, seed=1)
    packed = mx4._pack("test", up, ups, E, None)
    for T in (1, 15, 16):
        ids, _ = route(T, E, K, seed=T)
        groups = group_rows(ids, E)
        x = torch.randn(T, H, generator=gen(T), device="cuda").bfloat16()
        a, b = product(x, packed, groups, 2 * I, H), product(mx4.mx4_rows(x), packed, groups, 2 * I, H)
        assert (a - b).abs().max() <= 24 * STEP * 40


def test_strided_and_empty(hip):
    """x and out inside larger tensors; all pairs of one expert; no pair at all."""
    E, H, I, T, K = 5, 96, 64, 33, 2
    up, ups = weights(E, 2 * I, H, seed=1)
    down, downs = weights(E, H, I, seed=2)
    layer = Mx4Experts(up, ups, down, downs, max_tokens=64, top_k=K)
    big = torch.full((T, 160), float("nan"), device="cuda").bfloat16()
    x = big[:, 32:128]
    x.copy_(torch.randn(T, H, generator=gen(9), device="cuda"))
    _, wts = route(T, E, K, seed=2)
    out = torch.full((T + 1, 120), 7.0, device="cuda")
    for fill in (2, E, -1):
        ids = torch.full((T, K), fill, dtype=torch.int32, device="cuda")
        layer(x, ids, wts, out=out[:T, :H])
        assert torch.equal(out[:T, :H], layer(x.contiguous(), ids, wts, out=torch.empty(T, H, device="cuda")))
        assert (out[:, H:] == 7).all() and (out[T] == 7).all()
        if fill != 2:
            assert (out[:T, :H] == 0).all()


def test_layer_in_a_graph(hip):
    """Captured once, replayed with other routes: the grid covers any raggedness."""
    E, H, I, T, K = 9, 256, 96, 40, 3
    up, ups = weights(E, 2 * I, H, seed=1)
    down, downs = weights(E, H, I, seed=2)
    layer, eager = (Mx4Experts(up, ups, down, downs, max_tokens=T, top_k=K) for _ in range(2))
    x = torch.randn(T, H, generator=gen(1), device="cuda").bfloat16()
    ids, wts = route(T, E, K, seed=0)
    out = torch.empty_like(x)
    layer(x, ids, wts, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(x, ids, wts, out=out)
    for s in range(4):
        x.copy_(torch.randn(T, H, generator=gen(s), device="cuda"))
        i2, w2 = route(T, E, K, seed=s + 5, none=0.2 * s)
        ids.copy_(i2 if s != 3 else torch.zeros_like(i2))
        wts.copy_(w2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager(x, ids, wts))


def test_refused(hip):
    up, ups = weights(3, 128, 96, seed=1)
    down, downs = weights(3, 96, 64, seed=2)
    layer = Mx4Experts(up, ups, down, downs, max_tokens=4, top_k=2)
    x = torch.zeros(4, 96, device="cuda").bfloat16()
    ids, wts = route(4, 3, 2, seed=1)
    for args in ((x.float(), ids, wts), (x[:, :64], ids, wts), (torch.cat((x, x)), ids, wts), (x, ids.long(), wts),
                 (x, ids[:, :1], wts), (x, ids, wts.double()), (x, ids[:3], wts), (x.cpu(), ids, wts)):
        with pytest.raises(ValueError):
            layer(*args)
    for args in ((up, ups, down[:2], downs[:2]), (up, ups[:, :64], down, downs), (up[:, :96], ups[:, :96], down, downs),
                 (up[0], ups[0], down, downs)):
        with pytest.raises(ValueError):
            Mx4Experts(*args, max_tokens=4, top_k=2)
    with pytest.raises(ValueError):
        Mx4Experts(up, ups, down, downs, max_tokens=0, top_k=2)
    groups = RowGroups(4, 2, 3)
    group_rows(ids, 3, out=groups)
    with pytest.raises(_lib.HiRocmError):  # a half of 48 columns
        product(x, mx4._pack("test", up[:, :96].contiguous(), ups[:, :96].contiguous(), 3, None), groups, 96, 96, swiglu=True)
    assert combine(torch.zeros(8, 96, device="cuda"), groups, wts).shape == (4, 96)

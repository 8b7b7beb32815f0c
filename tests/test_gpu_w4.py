"""Products with 4-bit weights against (q - z) s x in 64 bits.

An output is a sum over groups of s (d - (16 + z) e), d = sum x (16 + q) and
e = sum x over the group in f32.  A sum of G terms is off by at most G eps
times the sum of their magnitudes, so a group by (G + 4) eps s sum |x| (32 + q
+ z), and the sum over K / G groups adds K / G eps of the groups' magnitudes.
That bounds every output; as the errors of random inputs do not conspire, the
whole is held to NORM in the 2-norm too (eps sqrt(32) 24 / 4.6 is 2e-6 of a
group's own size at its last term, and about a sixth of that over the sum)."""
import numpy as np
import pytest
import torch

from hi_amd import _lib
from hi_amd.w4 import W4Linear, quantize_w4

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
NORM = 2e-6


def weights(n, k, group, sdtype, zeros, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = ((torch.rand(n, k // group, generator=g, device="cuda") - 0.3) * 0.02).to(sdtype)
    z = torch.randint(0, 16, (n, k // group), generator=g, device="cuda").to(sdtype) if zeros else None
    return q, s, z


def exact(x, q, s, z, group, bias=None):
    """The products and the bound above."""
    n, k = q.shape[0], q.shape[1] * 2
    qq = torch.stack((q & 15, q >> 4), 2).view(n, k).double().cpu()
    ss = s.double().cpu().repeat_interleave(group, 1)
    zz = (z.double().cpu() if z is not None else torch.full(s.shape, 8.0, dtype=torch.float64)).repeat_interleave(group, 1)
    xx = x.double().cpu()
    y = xx @ ((qq - zz) * ss).t()
    size = xx.abs() @ (ss.abs() * (32 + qq + zz)).t()
    tol = (group + 4 + k // group) * EPS * size
    if bias is not None:
        y = y + bias.double().cpu()
        tol = tol + 2 * EPS * y.abs()
    return y, tol


def agree(got, y, tol):
    """Within the bound; a bf16 result is the rounding of a value within it."""
    if got.dtype == torch.bfloat16:
        lo, hi = (y - tol).float().bfloat16(), (y + tol).float().bfloat16()
        assert ((got.cpu() >= lo) & (got.cpu() <= hi)).all()
        return
    d = (got.double().cpu() - y).abs()
    assert (d <= tol).all(), (d - tol).max()
    if y.numel() >= 256:
        assert d.norm() <= NORM * y.norm(), d.norm() / y.norm()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("sdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,n,groups", [(1, 1, 1), (1, 1000, 5), (3, 17, 9), (16, 64, 33), (17, 100, 4), (33, 48, 7),
                                           (64, 130, 16), (65, 20, 3), (200, 33, 2)])
def test_products(hip, group, sdtype, zeros, rows, n, groups):
    k = group * groups
    q, s, z = weights(n, k, group, sdtype, zeros, seed=rows * 7 + n)
    x = torch.randn(rows, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(rows)).bfloat16()
    bias = torch.randn(n, device="cuda")
    lin = W4Linear(q, s, z, bias=bias if rows % 2 else None)
    y, tol = exact(x, q, s, z, group, lin.bias)
    agree(lin(x), y, tol)
    agree(lin(x, dtype=torch.bfloat16), y, tol)


@pytest.mark.parametrize("rows,n,k", [(1, 151936, 4096), (2, 40000, 2048), (48, 16384, 4096), (5, 513, 16384)])
def test_large(hip, rows, n, k):
    q, s, z = weights(n, k, 64, torch.bfloat16, True, seed=n)
    x = torch.randn(rows, k, device="cuda").bfloat16()
    got = W4Linear(q, s, z)(x)
    at = torch.randint(0, n, (300,), device="cuda").unique()
    at = torch.cat((at, torch.tensor([0, n - 1], device="cuda")))
    y, tol = exact(x, q[at], s[at], z[at], 64)
    agree(got[:, at], y, tol)


def test_rows_do_not_mix(hip):
    """A row's bits are the same whatever the other rows hold, NaN and inf
    among them, as long as the same kernel takes the call."""
    q, s, z = weights(96, 640, 32, torch.float32, True, seed=1)
    lin = W4Linear(q, s, z)
    x = torch.randn(16, 640, device="cuda").bfloat16()
    y = lin(x)
    x2 = x.clone()
    x2[3], x2[4, 0], x2[5, 639] = float("nan"), float("inf"), float("nan")
    y2 = lin(x2)
    keep = [i for i in range(16) if i not in (3, 4, 5)]
    assert torch.equal(y[keep], y2[keep])
    assert y2[[3, 4, 5]].isnan().all()
    assert torch.equal(lin(x), y)


def test_padding_stays_out(hip):
    """k that ends inside a block and n inside a tile: what lies behind the
    inputs (NaN) and the outputs (a mark) is neither used nor written."""
    q, s, z = weights(21, 160, 32, torch.bfloat16, False, seed=2)
    big = torch.full((5, 320), float("nan"), device="cuda").bfloat16()
    x = big[:, :160]
    x.copy_(torch.randn(5, 160, device="cuda"))
    out = torch.full((5, 40), 77.0, device="cuda")
    W4Linear(q, s, z)(x, out=out[:, :21])
    y, tol = exact(x, q, s, z, 32)
    agree(out[:, :21].clone(), y, tol)
    assert (out[:, 21:] == 77.0).all()


def test_extremes(hip):
    """q at both ends, zero scales, large and tiny activations."""
    q = torch.tensor([[0x00] * 64, [0xff] * 64, [0x0f] * 64, [0x88] * 64], dtype=torch.uint8, device="cuda")
    s = torch.tensor([[1.0], [0.0], [2.0 ** -60], [1.0]], device="cuda")
    lin = W4Linear(q, s)
    for scale in (1.0, 2.0 ** 100, 2.0 ** -100):
        x = (torch.randn(2, 128, device="cuda") * scale).bfloat16()
        y, tol = exact(x, q, s, None, 128)
        d = (lin(x).double().cpu() - y).abs()
        assert (d <= tol + 2.0 ** -149).all()  # (2^-160 is less than f32 holds)
    assert (lin(x)[:, 1] == 0).all() and (lin(x)[:, 3] == 0).all()


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 128])
def test_quantize(hip, symmetric, group):
    g = torch.Generator(device="cuda").manual_seed(5)
    w = torch.randn(40, 512, generator=g, device="cuda") + (0.0 if symmetric else 0.5)
    w[3] = 0.0
    q, s, z = quantize_w4(w, group, symmetric)
    back = W4Linear(q, s, z)(torch.eye(512, device="cuda").bfloat16()).t()
    # the nearest of the 16 values that the scale and zero give
    ss = s.double().repeat_interleave(group, 1)
    zz = z.double().repeat_interleave(group, 1) if z is not None else 8.0
    best = torch.stack([((v - zz) * ss - w.double()).abs() for v in range(16)]).amin(0)
    assert ((back.double() - w.double()).abs() <= best + (group + 4) * EPS * ss * 48 + EPS * w.abs()).all()


def test_streams_and_graph(hip):
    q, s, z = weights(300, 512, 32, torch.bfloat16, True, seed=3)
    lin = W4Linear(q, s, z)
    x = torch.randn(4, 512, device="cuda").bfloat16()
    want = lin(x)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    got = lin(x, stream=st)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    out = torch.empty(4, 300, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        lin(x, out=out)
    for i in range(3):
        x.copy_(torch.randn(4, 512, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, lin(x))


def test_refusals(hip):
    q, s, z = weights(32, 128, 32, torch.float32, True, seed=4)
    for bad in (lambda: W4Linear(q.int(), s), lambda: W4Linear(q, s[:16]), lambda: W4Linear(q, s.half()),
                lambda: W4Linear(q, s, z.bfloat16()), lambda: W4Linear(q, s, z[:, :2]), lambda: W4Linear(q, s.cpu()),
                lambda: W4Linear(q.cpu(), s.cpu()), lambda: W4Linear(q, s, bias=torch.zeros(31, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_lib.HiRocmError):  # groups of 16
        W4Linear(q, torch.ones(32, 8, device="cuda"))
    lin = W4Linear(q, s, z)
    x = torch.zeros(2, 128, device="cuda").bfloat16()
    for bad in (lambda: lin(x.float()), lambda: lin(x[:, :64]), lambda: lin(x[0]), lambda: lin(x[:0]),
                lambda: lin(x, out=torch.zeros(2, 31, device="cuda")), lambda: lin(x.cpu()),
                lambda: lin(x, out=torch.zeros(2, 32, device="cuda", dtype=torch.float16))):
        with pytest.raises(ValueError):
            bad()
    wide = torch.zeros(2, 256, device="cuda").bfloat16()
    with pytest.raises(_lib.HiRocmError):  # rows that do not start on 16 bytes
        lin(wide[:, 1:129])


def test_packing_on_another_stream(hip, new_stream):
    """The quantised weight may be freed as soon as the call returns: its memory
    serves no new tensor before the packing, on a busy stream, has read it."""
    n, k = 4096, 1024
    q, s, z = weights(n, k, 32, torch.float32, True, seed=6)
    x = torch.randn(2, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(6)).bfloat16()
    want = W4Linear(q, s, z)(x)
    torch.cuda.synchronize()
    st = new_stream()
    with torch.cuda.stream(st):
        torch.cuda._sleep(200_000_000)
    lin = W4Linear(q, s, z, stream=st)
    busy = not st.query()
    old = {t.data_ptr() for t in (q, s, z)}
    shapes = [(t.shape, t.dtype) for t in (q, s, z)]
    del q, s, z
    new = [torch.full(shape, 3, dtype=dtype, device="cuda") for shape, dtype in shapes]
    assert busy and not old & {t.data_ptr() for t in new}
    torch.cuda.synchronize()
    assert torch.equal(lin(x), want)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("sdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("rows,n,blocks", [
    # one row: one tile of outputs a workgroup, two, four; k in one pass and in several
    (1, 4000, 20), (1, 8100, 12), (1, 4300, 20), (1, 4300, 37), (1, 8300, 5), (1, 8300, 13), (1, 8300, 35),
    # up to 16 rows, the same
    (5, 4000, 20), (5, 8100, 12), (8, 4300, 20), (16, 8300, 5), (9, 8300, 13), (9, 8300, 35),
    # more, 16 rows a workgroup and 32
    (40, 2000, 5), (40, 4300, 13), (24, 8300, 5), (40, 8300, 13), (20, 4300, 20), (20, 8300, 35)])
def test_every_split(hip, group, sdtype, zeros, rows, n, blocks):
    """Each way to share outputs, rows and k among workgroups and waves; the
    last block of 128 inputs holds one group."""
    k = (blocks - 1) * 128 + group
    q, s, z = weights(n, k, group, sdtype, zeros, seed=n + blocks)
    x = torch.randn(rows, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(rows)).bfloat16()
    bias = torch.randn(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(n)) if rows % 2 else None
    lin = W4Linear(q, s, z, bias=bias)
    got, half = lin(x), lin(x, dtype=torch.bfloat16)
    at = torch.cat((torch.arange(0, n, 29), torch.arange(n - 20, n))).cuda().unique()
    y, tol = exact(x, q[at], s[at], z[at] if zeros else None, group, None if bias is None else bias[at])
    agree(got[:, at], y, tol)
    agree(half[:, at], y, tol)

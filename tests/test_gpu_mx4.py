"""Microscaled 4-bit floating point against its definition in 64 bits.

Rounding and values are exact.  A product's terms (code times code times powers
of two) are exact in f32; a sum over k / 32 blocks and the waves' shares of it
rounds at most k / 32 + 8 times, each within a step of 2^-23 of the magnitudes
summed (a step, not half, as the matrix cores need not round to nearest).  As
those errors do not conspire, the whole is held to NORM in the 2-norm too:
sqrt(64) steps at the largest k here."""
import pytest
import torch

from hi_amd import _lib, mx4
from hi_amd.mx4 import Mx4Linear, dequantize_mx4, mx4_rows, quantize_mx4
from oracle import mx4_oracle as O

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -23
NORM = 2e-6


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def weight(n, k, seed):
    """Random codes and scales: products of different size in a sum."""
    g = gen(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.randint(115, 125, (n, k // 32), generator=g, device="cuda", dtype=torch.uint8)
    return codes, scales


def exact(x, codes, scales, bias=None):
    xx, ww = O.rounded(x), O.values(codes, scales)
    y, size = xx @ ww.t(), xx.abs() @ ww.abs().t()
    tol = (x.shape[1] // 32 + 8) * STEP * size
    if bias is not None:
        y = y + bias.double().cpu()
        tol = tol + STEP * y.abs()
    return y, tol


def agree(got, y, tol):
    got = got.cpu()
    if got.dtype == torch.bfloat16:
        lo, hi = (y - tol).float().bfloat16(), (y + tol).float().bfloat16()
        assert ((got >= lo) & (got <= hi)).all()
        return
    d = (got.double() - y).abs()
    assert (d <= tol).all(), (d - tol).max()
    if y.numel() >= 256:
        assert d.norm() <= NORM * y.norm(), d.norm() / y.norm()


def same_rounding(x):
    codes, scales = quantize_mx4(x)
    want, s = O.quantize(x)
    assert torch.equal(scales.cpu(), s)
    assert torch.equal(codes.cpu(), O.pack_nibbles(want))
    v = O.values(codes, scales)
    for dtype in (torch.float32, torch.bfloat16):
        got = dequantize_mx4(codes, scales, dtype=dtype).cpu()
        w = v.to(dtype)  # (each has two bits: exact, or infinite beyond the type)
        assert torch.equal(got.isnan(), w.isnan())
        assert torch.equal(got.nan_to_num(nan=0.0), w.nan_to_num(nan=0.0))
        assert torch.equal(torch.signbit(got)[~w.isnan()], torch.signbit(w)[~w.isnan()])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 512), (3, 64), (2, 544), (5, 1184), (17, 96), (130, 1024), (4097, 32),
                                    (2, 20000 // 32 * 32)])
def test_rounding(hip, dtype, rows, k):
    x = torch.randn(rows, k, generator=gen(rows + k), device="cuda")
    x *= torch.exp(torch.randn(rows, 1, generator=gen(k), device="cuda") * 4)
    same_rounding(x.to(dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rounding_at_borders(hip, dtype):
    """Blocks of every exponent, subnormal ones too: values at and next to the
    borders between codes, the largest value of each mantissa, zeros."""
    m = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0])
    step = torch.finfo(dtype).eps
    m = torch.cat((m, m * (1 + step), m * (1 - step / 2), -m))  # [64]
    rows = []
    for e in range(-152, 128):
        for top in (4.0, 6.0, 7.0, 7.96875):
            r = torch.ldexp(torch.cat((m, torch.full((1,), top))).double(), torch.tensor(e - 2))
            rows.append(torch.stack((r[:31], r[31:62])).flatten())
            rows[-1] = torch.cat((r[:31], r[64:], r[31:62], r[64:]))
    x = torch.stack(rows).to(dtype)
    x = x[x.isfinite().all(1)]
    assert x.shape[0] > 1000
    same_rounding(x.cuda())
    same_rounding(torch.zeros(3, 64, dtype=dtype, device="cuda"))
    same_rounding(-torch.zeros(3, 64, dtype=dtype, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_blocks_that_are_not_finite(hip, dtype):
    x = torch.randn(8, 96, generator=gen(1), device="cuda").to(dtype)
    x[1, 3], x[2, 40], x[3, 95], x[4, 64] = float("inf"), float("nan"), float("-inf"), -float("nan")
    same_rounding(x)
    codes, scales = quantize_mx4(x)
    assert (scales == 255).sum() == 4


def test_every_code_and_scale(hip):
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")[:, None].expand(256, 16 * 256).contiguous()
    scales = torch.arange(256, dtype=torch.uint8, device="cuda")[None].expand(256, 256).contiguous()
    v = O.values(codes, scales)
    for dtype in (torch.float32, torch.bfloat16):
        got, w = dequantize_mx4(codes, scales, dtype=dtype).cpu(), v.to(dtype)
        assert torch.equal(got.isnan(), w.isnan())
        assert torch.equal(got.nan_to_num(nan=0.0), w.nan_to_num(nan=0.0))


def test_rounding_strides(hip):
    big = torch.full((7, 256), float("nan"), device="cuda")
    big[:, 32:128] = torch.randn(7, 96, generator=gen(5), device="cuda")
    for view in (big[:, 32:128], big[::2, 32:128]):
        same_rounding(view)
    codes, scales = quantize_mx4(big[:, 32:128])
    out = torch.full((7, 160), 77.0, device="cuda")
    dequantize_mx4(codes, scales, out=out[:, 32:128])
    assert (out[:, :32] == 77).all() and (out[:, 128:] == 77).all()
    assert torch.equal(out[:, 32:128].cpu(), O.values(codes, scales).float())


@pytest.mark.parametrize("rows", [1, 2, 5, 16, 17, 33, 64, 65, 130, 257])
@pytest.mark.parametrize("n,k", [(1, 32), (16, 128), (17, 96), (63, 160), (100, 512), (64, 544), (130, 1184), (300, 2048),
                                 (1000, 64), (513, 640)])
def test_products(hip, rows, n, k):
    codes, scales = weight(n, k, seed=n + k)
    x = torch.randn(rows, k, generator=gen(rows), device="cuda").bfloat16()
    bias = torch.randn(n, generator=gen(n), device="cuda") if rows % 2 else None
    lin = Mx4Linear(codes, scales, bias)
    y, tol = exact(x, codes, scales, bias)
    agree(lin(x), y, tol)
    agree(lin(x, dtype=torch.bfloat16), y, tol)
    agree(lin(mx4_rows(x)), y, tol)


@pytest.mark.parametrize("rows,n,k", [(1, 151936, 4096), (8, 40000, 2048), (320, 16384, 4096), (2048, 4096, 4096),
                                      (5, 513, 16384), (1000, 5000, 1184), (4096, 1024, 512)])
def test_large(hip, rows, n, k):
    codes, scales = weight(n, k, seed=n)
    x = torch.randn(rows, k, generator=gen(rows), device="cuda").bfloat16()
    got = Mx4Linear(codes, scales)(x)
    c = torch.cat((torch.randint(0, n, (300,), device="cuda"), torch.tensor([0, n - 1], device="cuda"))).unique()
    r = torch.cat((torch.randint(0, rows, (50,), device="cuda"), torch.tensor([0, rows - 1], device="cuda"))).unique()
    y, tol = exact(x[r], codes[c], scales[c])
    agree(got[r][:, c], y, tol)


@pytest.mark.parametrize("k", [32, 96, 256, 384, 512, 544, 896, 1184, 1664])
@pytest.mark.parametrize("rows,n", [(130, 16400), (250, 16380), (310, 16384), (509, 16385), (2048, 4097), (33, 70001)])
def test_tiles(hip, rows, n, k):
    """Every size of tile, tiles that end inside the places or the weight's last
    rows, and every number of steps behind whole quads: the last rows and columns
    and some between."""
    codes, scales = weight(n, k, seed=k)
    x = torch.randn(rows, k, generator=gen(rows), device="cuda").bfloat16()
    bias = torch.randn(n, generator=gen(n), device="cuda")
    lin = Mx4Linear(codes, scales, bias)
    c = torch.cat((torch.randint(0, n, (200,), generator=gen(1), device="cuda"), torch.arange(n - 70, n, device="cuda"))).unique()
    r = torch.cat((torch.randint(0, rows, (40,), generator=gen(2), device="cuda"),
                   torch.arange(rows - 33, rows, device="cuda"))).unique()
    y, tol = exact(x[r], codes[c], scales[c], bias[c])
    for dtype in (torch.float32, torch.bfloat16):
        agree(lin(x, dtype=dtype)[r][:, c], y, tol)


@pytest.mark.parametrize("k", [1056, 1568, 2048, 2592, 3104, 3680, 4640, 8224])
@pytest.mark.parametrize("rows,n", [(300, 1001), (300, 2050), (330, 4090), (190, 70), (500, 4001)])
def test_narrow_tiles(hip, rows, n, k):
    """Few columns, whose tiles share out k: stretches of different lengths, of no
    quad, and ones that end inside a quad."""
    codes, scales = weight(n, k, seed=k)
    x = torch.randn(rows, k, generator=gen(rows), device="cuda").bfloat16()
    bias = torch.randn(n, generator=gen(n), device="cuda")
    lin = Mx4Linear(codes, scales, bias)
    c = torch.cat((torch.randint(0, n, (200,), generator=gen(1), device="cuda"), torch.arange(n - 70, n, device="cuda"))).unique()
    r = torch.cat((torch.randint(0, rows, (60,), generator=gen(2), device="cuda"),
                   torch.arange(rows - 65, rows, device="cuda"))).unique()
    y, tol = exact(x[r], codes[c], scales[c], bias[c])
    for dtype in (torch.float32, torch.bfloat16):
        agree(lin(x, dtype=dtype)[r][:, c], y, tol)


@pytest.mark.parametrize("k", [32, 160, 512, 1184, 2080, 4096])
@pytest.mark.parametrize("rows,n", [(17, 48), (40, 1000), (100, 130), (500, 65), (1999, 48), (64, 2048), (30, 8190)])
def test_more_rows_without_a_workspace(hip, rows, n, k):
    """Rows rounded by the workgroups that multiply them, whatever their number: the
    result of rows rounded beforehand, up to the order of the sums."""
    codes, scales = weight(n, k, seed=n + k)
    x = torch.randn(rows, k, generator=gen(rows), device="cuda").bfloat16()
    bias = torch.randn(n, generator=gen(n), device="cuda")
    lin = Mx4Linear(codes, scales, bias)
    r = torch.cat((torch.randint(0, rows, (40,), generator=gen(2), device="cuda"),
                   torch.arange(max(rows - 20, 0), rows, device="cuda"))).unique()
    y, tol = exact(x[r], codes, scales, bias)
    for given in (x, mx4_rows(x)):
        for dtype in (torch.float32, torch.bfloat16):
            agree(lin(given, dtype=dtype)[r], y, tol)


@pytest.mark.parametrize("rows,n", [(7, 96), (16, 96), (40, 96), (200, 96), (130, 16384), (520, 16384), (2000, 4096)])
def test_rows_do_not_mix(hip, rows, n):
    """A row's bits are the same whatever the other rows hold; a row with an
    infinity or NaN gives NaN."""
    codes, scales = weight(n, 640, seed=1)
    lin = Mx4Linear(codes, scales)
    x = torch.randn(rows, 640, generator=gen(2), device="cuda").bfloat16()
    y = lin(x)
    x2 = x.clone()
    x2[3], x2[4, 0], x2[5, 639] = float("nan"), float("inf"), float("nan")
    y2 = lin(x2)
    keep = [i for i in range(rows) if i not in (3, 4, 5)]
    assert torch.equal(y[keep], y2[keep])
    assert y2[[3, 4, 5]].isnan().all()
    assert torch.equal(lin(x), y)


@pytest.mark.parametrize("rows,n", [(3, 40), (70, 40), (300, 40), (300, 1000)])
def test_scales_at_their_ends(hip, rows, n):
    """Weights of NaN blocks, of the smallest and largest scales, and of zeros."""
    codes, scales = weight(n, 192, seed=3)
    scales[7, 2] = 255
    scales[8], scales[9] = 0, 250
    codes[10] = 0
    scales[10] = 254
    x = torch.randn(rows, 192, generator=gen(4), device="cuda").bfloat16()
    x[1] = 0
    x[2] *= 2.0 ** -110
    got = Mx4Linear(codes, scales)(x)
    y, tol = exact(x, codes, scales)
    # Every partial sum is at most the sum of the magnitudes.  Where that passes
    # f32's largest, partial sums of both signs may be infinite and their sum NaN.
    fits = ~(tol / ((192 // 32 + 8) * STEP) > torch.finfo(torch.float32).max)
    assert (~fits).sum() <= rows
    assert torch.equal(got.cpu().isnan()[fits], y.isnan()[fits]) and y.isnan().sum() == rows
    ok = ~y.isnan() & fits
    tiny = 2.0 ** -126 * 192  # results under the normal numbers may be flushed, a step at a time
    d = (got.double().cpu() - y).abs()
    assert (d[ok] <= (tol + tiny)[ok]).all()
    assert (got[:, 10] == 0).all()


@pytest.mark.parametrize("rows,n", [(5, 21), (40, 21), (300, 21), (300, 1013)])
def test_padding_stays_out(hip, rows, n):
    """k that ends inside a step and n inside a tile: what lies behind the
    inputs (NaN) and the outputs (a mark) is neither used nor written."""
    codes, scales = weight(n, 160, seed=2)
    big = torch.full((rows, 320), float("nan"), device="cuda").bfloat16()
    x = big[:, :160]
    x.copy_(torch.randn(rows, 160, generator=gen(6), device="cuda"))
    for dtype in (torch.float32, torch.bfloat16):
        for pad in (n + 19, n + 22):
            out = torch.full((rows + 1, pad), 77.0, device="cuda", dtype=dtype)
            Mx4Linear(codes, scales)(x, out=out[:rows, :n])
            y, tol = exact(x, codes, scales)
            agree(out[:rows, :n].clone(), y, tol)
            assert (out[:, n:] == 77).all() and (out[rows] == 77).all()


def test_rows_used_twice(hip):
    """Rows rounded once serve several weights, and are the call's own rounding."""
    x = torch.randn(90, 1056, generator=gen(7), device="cuda").bfloat16()
    rows = mx4_rows(x)
    for n in (64, 200):
        lin = Mx4Linear(*weight(n, 1056, seed=n))
        assert torch.equal(lin(rows), lin(x))
    f = torch.randn(3, 96, generator=gen(8), device="cuda")
    lin = Mx4Linear(*weight(33, 96, seed=9))
    codes, scales = quantize_mx4(f)
    y, tol = exact(O.values(codes, scales), *weight(33, 96, seed=9))
    agree(lin(mx4_rows(f)), y, tol)


def test_graph_replays(hip):
    """Captured calls (few rows, and rows rounded in a workspace) on new inputs,
    eager calls between the replays."""
    lin = Mx4Linear(*weight(1000, 512, seed=1))
    for rows in (3, 50, 400):
        x = torch.randn(rows, 512, generator=gen(rows), device="cuda").bfloat16()
        out = torch.empty(rows, 1000, device="cuda")
        lin(x, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lin(x, out=out)
        for i in range(4):
            x.copy_(torch.randn(rows, 512, generator=gen(i + 1), device="cuda"))
            out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            assert torch.equal(got, lin(x))


def test_other_stream(hip, new_stream):
    side = new_stream()
    codes, scales = weight(128, 256, seed=4)
    x = torch.randn(40, 256, generator=gen(1), device="cuda").bfloat16()
    torch.cuda.synchronize()
    lin = Mx4Linear(codes, scales, stream=side)
    got = lin(x, stream=side)
    c, s = quantize_mx4(x, stream=side)
    v = dequantize_mx4(c, s, stream=side)
    side.synchronize()
    y, tol = exact(x, codes, scales)
    agree(got, y, tol)
    assert torch.equal(v.cpu(), O.rounded(x).bfloat16())


def test_refused(hip):
    codes, scales = weight(32, 64, seed=1)
    lin = Mx4Linear(codes, scales)
    x = torch.zeros(4, 64, device="cuda").bfloat16()
    for bad in (x.float(), x[:, :32], x[0], x.t(), x[:0], torch.zeros(4, 128, device="cuda").bfloat16()[:, ::2]):
        with pytest.raises(ValueError):
            lin(bad)
    with pytest.raises(ValueError):
        lin(mx4_rows(torch.zeros(4, 96, device="cuda")))
    with pytest.raises(ValueError):
        lin(x, out=torch.zeros(4, 31, device="cuda"))
    with pytest.raises(ValueError):
        lin(x, out=torch.zeros(4, 32, device="cuda").half())
    for args in ((codes[:, :20], scales), (codes, scales[:, :1]), (codes.int(), scales), (codes.t(), scales.t()),
                 (codes.cpu(), scales.cpu()), (codes, scales, torch.zeros(31, device="cuda"))):
        with pytest.raises(ValueError):
            Mx4Linear(*args)
    for bad in (torch.zeros(2, 48, device="cuda"), torch.zeros(2, 64, device="cuda").half(), torch.zeros(64, device="cuda"),
                torch.zeros(2, 64)):
        with pytest.raises(ValueError):
            quantize_mx4(bad)
    with pytest.raises(_lib.HiRocmError) as e:  # rows that do not start on 16 bytes
        quantize_mx4(torch.zeros(2, 65, device="cuda")[:, 1:])
    assert e.value.status == _lib.ERR_UNSUPPORTED
    with pytest.raises(_lib.HiRocmError):
        lin(torch.zeros(4, 72, device="cuda").bfloat16()[:, 1:65])
    with pytest.raises(ValueError):
        mx4.mx4_rows(x, out=mx4.Mx4Rows(5, 64))

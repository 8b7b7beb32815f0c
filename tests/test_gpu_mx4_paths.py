"""Every way that a 4-bit linear layer's call is taken, against its definition in
64 bits; each case names the way it means, so that another choice of tiles cannot
leave one out unnoticed.

Bounds as in test_gpu_mx4.py: a sum rounds at most k / 32 + 8 times, each within
2^-23 of the magnitudes summed."""
import pytest
import torch

from hi_amd.mx4 import Mx4Linear, mx4_rows
from oracle import mx4_oracle as O
from test_mx4_paths import BF16, CASES, F32, FEW, path, workspace

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -23
CODES = {torch.float32: F32, torch.bfloat16: BF16}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def weight(n, k, seed):
    g = gen(seed)
    return (torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8),
            torch.randint(115, 125, (n, k // 32), generator=g, device="cuda", dtype=torch.uint8))


def some(size, last, count, seed):
    """Some of [0, size), the last ones among them."""
    return torch.cat((torch.randint(0, size, (count,), generator=gen(seed), device="cuda"),
                      torch.arange(max(size - last, 0), size, device="cuda"))).unique()


def agree(got, x, codes, scales, bias=None):
    """got [rows][n] of x and the weight, given in 32 bits or 16."""
    xx, ww = O.rounded(x), O.values(codes, scales)
    y, size = xx @ ww.t(), xx.abs() @ ww.abs().t()
    tol = (x.shape[1] // 32 + 8) * STEP * size
    if bias is not None:
        y = y + bias.double().cpu()
        tol = tol + STEP * y.abs()
    got = got.cpu()
    if got.dtype == torch.bfloat16:
        assert ((got >= (y - tol).float().bfloat16()) & (got <= (y + tol).float().bfloat16())).all()
    else:
        assert ((got.double() - y).abs() <= tol).all()


@pytest.mark.parametrize("rows,n,k,tile", CASES)
def test_definition(hip, rows, n, k, tile):
    """With a bias, in both types, of rows rounded beforehand and of bf16 ones."""
    codes, scales = weight(n, k, seed=k)
    x = torch.randn(rows, k, generator=gen(rows), device="cuda").bfloat16()
    bias = torch.randn(n, generator=gen(n), device="cuda")
    lin = Mx4Linear(codes, scales, bias)
    assert path(rows, n, k)[0] == tile
    r, c = some(rows, 33, 40, 1), some(n, 70, 200, 2)
    for given in (mx4_rows(x), x):
        for dtype in (torch.float32, torch.bfloat16):
            agree(lin(given, dtype=dtype)[r][:, c], x[r], codes[c], scales[c], bias[c])


@pytest.mark.parametrize("rows,n,k,tile", [c for c in CASES if c[0] > 2])
def test_scales_at_their_ends(hip, rows, n, k, tile):
    """Weights of a NaN block, of the smallest and largest scales, and of zeros; rows of
    zeros and of next to nothing."""
    codes, scales = weight(n, k, seed=3)
    scales[7, 2] = 255
    scales[8], scales[9] = 0, 250
    codes[10] = 0
    scales[10] = 254
    x = torch.randn(rows, k, generator=gen(4), device="cuda").bfloat16()
    x[1] = 0
    x[2] *= 2.0 ** -110
    r, c = some(rows, 33, 40, 1), torch.cat((torch.arange(16, device="cuda"), some(n, 20, 40, 2))).unique()
    r = torch.cat((torch.arange(3, device="cuda"), r)).unique()
    xx, ww = O.rounded(x[r]), O.values(codes[c], scales[c])
    y, size = xx @ ww.t(), xx.abs() @ ww.abs().t()
    tol = (k // 32 + 8) * STEP * size + 2.0 ** -126 * k  # (results under the normal numbers may be flushed)
    fits = ~(size > torch.finfo(torch.float32).max)  # partial sums beyond f32 may be infinite, and NaN of both signs
    for given in (mx4_rows(x), x):
        got = Mx4Linear(codes, scales)(given)
        part = got[r][:, c].double().cpu()
        assert torch.equal(part.isnan()[fits], y.isnan()[fits]) and y[:, 7].isnan().all() and y.isnan().sum() == len(r)
        ok = ~y.isnan() & fits
        assert ((part - y).abs()[ok] <= tol[ok]).all()
        assert (got[:, 10] == 0).all() and got[:, 7].isnan().all() and not got[:, 11:].isnan().any()


@pytest.mark.parametrize("rows,n,k,tile", CASES)
def test_what_lies_around(hip, rows, n, k, tile):
    """NaN behind the inputs, a mark behind the outputs: neither used nor written, for
    rows of the result on 16 bytes and elsewhere."""
    codes, scales = weight(n, k, seed=2)
    big = torch.full((rows, k + 96), float("nan"), device="cuda").bfloat16()
    x = big[:, :k]
    x.copy_(torch.randn(rows, k, generator=gen(6), device="cuda"))
    lin = Mx4Linear(codes, scales)
    r, c = some(rows, 33, 20, 1), some(n, 70, 40, 2)
    for given in (mx4_rows(x), x):
        for dtype in (torch.float32, torch.bfloat16):
            for stride in ((n + 16) // 8 * 8, (n + 16) | 1):
                out = torch.full((rows + 1, stride), 77.0, device="cuda", dtype=dtype)
                lin(given, out=out[:rows, :n])
                assert (out[:, n:] == 77).all() and (out[rows] == 77).all()
                agree(out[r][:, c], x[r], codes[c], scales[c])


@pytest.mark.parametrize("rows,n,k", [(50, 1000, 4640), (300, 16384, 512), (17, 48, 4128), (400, 2050, 1184)])
def test_graph_with_a_workspace(hip, rows, n, k):
    """Rows rounded in a workspace that the captured call allocates: replays on new
    inputs, eager calls, whose workspace is another, between them."""
    assert workspace(rows, n, k) > 0
    lin = Mx4Linear(*weight(n, k, seed=1))
    x = torch.randn(rows, k, generator=gen(rows), device="cuda").bfloat16()
    out = torch.empty(rows, n, device="cuda")
    lin(x, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lin(x, out=out)
    for i in range(4):
        x.copy_(torch.randn(rows, k, generator=gen(i + 1), device="cuda"))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, lin(x)) and torch.equal(got, lin(mx4_rows(x)))


@pytest.mark.parametrize("rows,n,k,dtype,past", [
    (320, 4093, 512, torch.bfloat16, False), (320, 4096, 512, torch.bfloat16, False), (321, 16384, 544, torch.bfloat16, True),
    (321, 16387, 544, torch.float32, True), (8190, 4096, 256, torch.float32, False), (8190, 4099, 256, torch.float32, False),
    (8190, 16384, 160, torch.bfloat16, True), (4094, 16389, 160, torch.float32, True)])
def test_stores(hip, rows, n, k, dtype, past):
    """Results stored past the caches and not, whole rows and ragged ones, at the right
    places and nowhere else."""
    codes, scales = weight(n, k, seed=n)
    x = torch.randn(rows, k, generator=gen(rows), device="cuda").bfloat16()
    tile, got = path(rows, n, k, out_dtype=CODES[dtype])
    assert tile[0] > 16 and got is past
    lin, pad = Mx4Linear(codes, scales), 16 if n % 8 == 0 else 13
    out = torch.full((rows + 1, n + pad), 77.0, dtype=dtype, device="cuda")
    lin(mx4_rows(x), out=out[:rows, :n])
    assert (out[:, n:] == 77).all() and (out[rows] == 77).all()
    r, c = some(rows, 33, 40, 1), some(n, 70, 200, 2)
    agree(out[r][:, c], x[r], codes[c], scales[c])
    assert torch.equal(lin(mx4_rows(x), dtype=dtype), out[:rows, :n])

"""Every way that a 4-bit linear layer's call is taken, against its definition in
64 bits; each case names the way it means, so that another choice of tiles cannot
leave one out unnoticed.

Bounds as in test_gpu_mx4.py: a sum rounds at most k / 32 + 8 times, each within
2^-23 of the magnitudes summed."""
import pytest
import torch

from hi_amd import _lib
from hi_amd.mx4 import Mx4Linear, mx4_rows
from oracle import mx4_oracle as O
from test_mx4_paths import BF16, F32, MX4, path

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

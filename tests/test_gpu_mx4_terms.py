"""The type of a token's terms in the 4-bit expert layer.

A term alone is the layer's f32 result where its weight is 1 and the others' 0
(sums with zeros are exact).  Sums of K weighted terms round 2 K times in f32 at
most; a term in bf16 is off by up to 2^-8 of itself, a bf16 result by 2^-8."""
import pytest
import torch

from hi_amd.mx4 import Mx4Experts, quantize_mx4

HALF32, HALF16 = 2.0 ** -24, 2.0 ** -8
gpu = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def weights(E, n, k, seed):
    codes, scales = quantize_mx4(torch.randn(E * n, k, generator=gen(seed), device="cuda") * k ** -0.5)
    return codes.view(E, n, k // 2), scales.view(E, n, k // 32)


def layer(E, H, I, T, K, **kw):
    return Mx4Experts(*weights(E, 2 * I, H, 1), *weights(E, H, I, 2), max_tokens=T, top_k=K, **kw)


def route(T, E, K, seed):
    g = gen(seed)
    ids = torch.rand(T, E, generator=g, device="cuda").topk(K, 1).indices.int()
    return ids, torch.rand(T, K, generator=g, device="cuda")


def inputs(T, E, H, K):
    return (torch.randn(T, H, generator=gen(T), device="cuda").bfloat16(), *route(T, E, K, seed=T + 1))


def terms_of(one, x, ids, K):
    """[T][K][H] float32."""
    alone = torch.eye(K, device="cuda")
    return torch.stack([one(x, ids, alone[s].expand(len(x), K).contiguous(),
                            out=torch.empty(x.shape, device="cuda")) for s in range(K)], 1)


SIZES = [(1, 4, 2, 64, 32), (5, 8, 3, 96, 64), (17, 60, 4, 320, 160), (200, 16, 4, 512, 224), (300, 4, 2, 1184, 352),
         (700, 8, 6, 256, 128)]


@gpu
@pytest.mark.parametrize("T,E,K,H,I", SIZES)
def test_a_result_has_one_rounding(hip, T, E, K, H, I):
    """A bf16 result is the f32 one rounded once, whatever is made of the layer first."""
    one = layer(E, H, I, T, K)
    x, ids, wts = inputs(T, E, H, K)
    got = one(x, ids, wts)
    full = one(x, ids, wts, out=torch.empty(T, H, device="cuda"))
    assert got.dtype == torch.bfloat16 and torch.equal(got, full.bfloat16())
    t, w = terms_of(one, x, ids, K).double(), wts.double()[:, :, None]
    d = (full.double() - (t * w).sum(1)).abs()
    assert (d <= 2 * K * HALF32 * (t.abs() * w).sum(1)).all()


@gpu
@pytest.mark.parametrize("T,E,K,H,I", SIZES)
def test_terms_in_bf16_when_asked_for(hip, T, E, K, H, I):
    """Each term rounded once, then the same sum, for either type of result."""
    full, half = layer(E, H, I, T, K), layer(E, H, I, T, K, terms=torch.bfloat16)
    x, ids, wts = inputs(T, E, H, K)
    t = terms_of(full, x, ids, K)
    assert torch.equal(terms_of(half, x, ids, K), t.bfloat16().float())
    t, w = t.bfloat16().double(), wts.double()[:, :, None]
    got = half(x, ids, wts, out=torch.empty(T, H, device="cuda"))
    assert ((got.double() - (t * w).sum(1)).abs() <= 2 * K * HALF32 * (t.abs() * w).sum(1)).all()
    assert torch.equal(half(x, ids, wts), got.bfloat16())


@gpu
@pytest.mark.parametrize("T", [6, 40, 300])
def test_terms_that_cancel(hip, T):
    """Weights for which two terms leave next to nothing of one column: what is left
    is as small as f32 leaves it, and with bf16 terms within their bound."""
    E, H, I, K = 9, 256, 96, 2
    full, half = layer(E, H, I, T, K), layer(E, H, I, T, K, terms=torch.bfloat16)
    x, ids, _ = inputs(T, E, H, K)
    t = terms_of(full, x, ids, K)
    at, row = t.abs().amin(1).argmax(1), torch.arange(T, device="cuda")  # a column where neither is small
    wts = torch.stack((torch.ones(T, device="cuda"), -t[row, 0, at] / t[row, 1, at]), 1).contiguous()
    terms, w = t.double(), wts.double()[:, :, None]
    want, size = (terms * w).sum(1), (terms * w).abs().sum(1)
    tol = 2 * K * HALF32 * size
    got = full(x, ids, wts).double()
    assert ((got - want).abs() <= tol + HALF16 * (want.abs() + tol)).all()
    assert (got[row, at].abs() <= 2 * K * 2 * HALF32 * size[row, at]).all()
    rough = half(x, ids, wts).double()
    bound = HALF16 * size + (1 + HALF16) * tol
    assert ((rough - want).abs() <= bound + HALF16 * (want.abs() + bound)).all()


def test_types_of_terms():
    up, s = torch.zeros(2, 64, 16, dtype=torch.uint8), torch.zeros(2, 64, 1, dtype=torch.uint8)
    down, d = torch.zeros(2, 32, 16, dtype=torch.uint8), torch.zeros(2, 32, 1, dtype=torch.uint8)
    for bad in (torch.float16, torch.float64, torch.uint8, None):
        with pytest.raises(ValueError, match="terms"):
            Mx4Experts(up, s, down, d, max_tokens=4, top_k=2, terms=bad)

"""Calls of the 4-bit layers as a program makes them: rows far apart in memory,
two streams at once, one layer for steps of different sizes, a token that is not
finite among others.  Results are equal to those of the same call alone."""
import pytest
import torch

from hi_amd.mx4 import Mx4Experts, Mx4Linear, dequantize_mx4, mx4_rows, quantize_mx4

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def weight(shape, k, seed):
    g = gen(seed)
    return (torch.randint(0, 256, (*shape, k // 2), generator=g, device="cuda", dtype=torch.uint8),
            torch.randint(118, 124, (*shape, k // 32), generator=g, device="cuda", dtype=torch.uint8))


def layer(E, H, I, tokens, top_k):
    up, ups = weight((E, 2 * I), H, seed=1)
    down, downs = weight((E, H), I, seed=2)
    return Mx4Experts(up, ups, down, downs, max_tokens=tokens, top_k=top_k)


def route(T, E, K, seed):
    ids = torch.rand(T, E, generator=gen(seed), device="cuda").topk(K, 1).indices.int()
    return ids, torch.rand(T, K, generator=gen(seed + 1), device="cuda")


@pytest.mark.parametrize("rows", [3, 20])
def test_rows_far_apart(hip, rows):
    """Rows whose offsets pass 32 bits, in bytes and in values."""
    k, n, far = 256, 96, 2 ** 32 // (rows - 1) // 64 * 64 + 64
    lin = Mx4Linear(*weight((n,), k, seed=1))
    x = torch.randn(rows, k, generator=gen(2), device="cuda").bfloat16()
    place = torch.empty((rows - 1) * far + k, dtype=torch.bfloat16, device="cuda")
    xs = place.as_strided((rows, k), (far, 1))
    xs.copy_(x)
    want = lin(x)
    assert torch.equal(lin(xs), want)
    assert torch.equal(lin(mx4_rows(xs)), want)
    codes, scales = quantize_mx4(xs)
    for a, b in zip((codes, scales), quantize_mx4(x)):
        assert torch.equal(a, b)
    back = dequantize_mx4(codes, scales)
    out = place.as_strided((rows, k), (far, 1))
    dequantize_mx4(codes, scales, out=out)
    assert torch.equal(out, back)
    out = place.as_strided((rows, n), (far, 1))
    lin(x, out=out)
    assert torch.equal(out, lin(x, dtype=torch.bfloat16))


def test_result_past_32_bits(hip):
    """A result of more than 2^31 values: its last rows and columns."""
    k, n, rows = 64, 151936, 14200
    codes, scales = weight((n,), k, seed=3)
    x = torch.randn(rows, k, generator=gen(4), device="cuda").bfloat16()
    got = Mx4Linear(codes, scales)(x, dtype=torch.bfloat16)
    tail = Mx4Linear(codes[-64:].contiguous(), scales[-64:].contiguous())(x[-50:].contiguous(), dtype=torch.bfloat16)
    # (two blocks of 32: one sum of two terms and exact products, whatever the tile)
    assert torch.equal(got[-50:, -64:], tail)


def test_two_streams_at_once(hip, new_stream):
    """One linear layer on two streams in turn, without waiting: the calls share
    weights alone."""
    lin = Mx4Linear(*weight((1000,), 4640, seed=5))
    a, b = new_stream(), new_stream()
    xs = [torch.randn(r, 4640, generator=gen(r), device="cuda").bfloat16() for r in (40, 300, 70, 513)]
    want = [lin(x) for x in xs]
    torch.cuda.synchronize()
    got = []
    for i in range(24):
        got.append((i % 4, lin(xs[i % 4], stream=(a, b)[i % 2 ^ (i // 4 & 1)])))
    torch.cuda.synchronize()
    for i, y in got:
        assert torch.equal(y, want[i])


def test_steps_of_different_sizes(hip):
    """What a large step left in a layer's buffers does not reach a small one's."""
    E, H, I, K = 12, 288, 160, 3
    one = layer(E, H, I, 700, K)
    for T in (700, 1, 16, 17, 333, 5, 700, 64):
        x = torch.randn(T, H, generator=gen(T), device="cuda").bfloat16()
        ids, wts = route(T, E, K, seed=T)
        assert torch.equal(one(x, ids, wts), layer(E, H, I, T, K)(x, ids, wts))


@pytest.mark.parametrize("T", [6, 40, 600])
def test_tokens_that_are_not_finite(hip, T):
    """Their own results are NaN, nobody else's change."""
    E, H, I, K = 6, 160, 96, 2
    one = layer(E, H, I, T, K)
    x = torch.randn(T, H, generator=gen(T), device="cuda").bfloat16()
    ids, wts = route(T, E, K, seed=T)
    want = one(x, ids, wts)
    bad = x.clone()
    bad[1, 3], bad[T - 1, H - 1], bad[T // 2, 40] = float("nan"), float("inf"), float("-inf")
    got = one(bad, ids, wts)
    rows = torch.zeros(T, dtype=torch.bool, device="cuda")
    rows[[1, T // 2, T - 1]] = True
    assert got[rows].isnan().all()
    assert torch.equal(got[~rows], want[~rows])

"""Symmetric 4-bit weights of 0 give 0, whatever x holds: a group's product and what
is taken off it round alike.  (With x of random values the two differed by a step of
f32 in one call of fifty where the second was 24 times a rounded sum.)"""
import pytest
import torch

from hi_amd.w4 import W4Linear

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("sdtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,n,k", [(1, 4, 128), (2, 40, 128), (16, 17, 1280), (33, 20, 256), (64, 48, 2048),
                                      (65, 20, 384), (1, 64, 16384)])
def test_weights_of_zero(hip, group, sdtype, rows, n, k):
    q = torch.randint(0, 256, (n, k // 2), generator=gen(1), device="cuda", dtype=torch.uint8)
    q[1::2] = 0x88
    s = (torch.rand(n, k // group, generator=gen(2), device="cuda") + 0.1).to(sdtype)
    lin = W4Linear(q, s)
    for seed in range(100):
        x = torch.randn(rows, k, generator=gen(seed), device="cuda")
        x *= torch.exp(torch.randn(k, generator=gen(seed + 1000), device="cuda") * (seed % 4)) * 2.0 ** (seed % 7 * 10 - 30)
        y = lin(x.bfloat16())
        assert (y[:, 1::2] == 0).all(), seed
        assert (y[:, ::2] != 0).any()


@pytest.mark.parametrize("group", [32, 128])
def test_groups_of_zero_add_nothing(hip, group):
    """One group with weights among groups of 0: the product of that group alone."""
    n, groups = 33, 8
    s = torch.rand(n, groups, generator=gen(3), device="cuda") + 0.1
    for at in range(groups):
        q = torch.full((n, groups * group // 2), 0x88, dtype=torch.uint8, device="cuda")
        part = torch.randint(0, 256, (n, group // 2), generator=gen(at), device="cuda", dtype=torch.uint8)
        q[:, at * group // 2:(at + 1) * group // 2] = part
        lin = W4Linear(q, s)
        alone = W4Linear(part, s[:, at:at + 1].contiguous())
        for seed in range(20):
            x = torch.randn(5, groups * group, generator=gen(seed), device="cuda").bfloat16()
            assert torch.equal(lin(x), alone(x[:, at * group:(at + 1) * group].contiguous()))

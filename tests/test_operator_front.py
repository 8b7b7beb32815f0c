"""Checks that the Python front ends of the beam, 4-bit and expert calls make
before anything reaches a device."""
import pytest
import torch

from hi_amd import beam, moe
from hi_amd.beam import BeamSearch, reorder_states
from hi_amd.w4 import W4Linear, quantize_w4


@pytest.mark.parametrize("rows,stride", [(4, 0), (4, 1), (4, 99), (8, 0), (2, 99)])
def test_rows_of_logits_that_overlap(rows, stride):
    """A view whose rows lie less than a vocabulary apart is refused: the
    kernels would read past it with any other stride."""
    bs = BeamSearch(4, 2, 100, device="cpu")
    memory = torch.zeros(100 + (rows - 1) * stride)
    logits = memory.as_strided((rows, 100), (stride, 1))
    with pytest.raises(ValueError, match="rows of logits overlap"):
        bs.select(logits, torch.zeros(rows))


def test_strides_of_logits_that_pass():
    """A single row's stride says nothing; rows may lie further apart.  (The
    next check is the device's.)"""
    one = BeamSearch(1, 1, 100, device="cpu")
    two = BeamSearch(1, 2, 100, device="cpu")
    for bs, logits in ((one, torch.zeros(100).expand(1, 100)), (one, torch.zeros(100).as_strided((1, 100), (7, 1))),
                       (two, torch.zeros(2, 100)), (two, torch.zeros(2, 132)[:, 16:116])):
        with pytest.raises(ValueError, match="needs CUDA tensors"):
            bs.select(logits, torch.zeros(logits.size(0)))


@pytest.mark.gpu
def test_tensors_and_stream_on_one_device(hip, new_stream, monkeypatch):
    """A call whose tensors are not on its stream's device (the current one, or
    the given stream's) is refused."""
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    w = torch.zeros(3, 64, 32, device="cuda").bfloat16()
    x = torch.zeros(4, 32, device="cuda").bfloat16()
    groups, layer = moe.group_rows(ids, 3), moe.MoeExperts(w, w[:, :32].contiguous(), 4, 2)
    q, s, _ = quantize_w4(torch.ones(16, 32, device="cuda"))
    lin, bs = W4Linear(q, s), BeamSearch(2, 2, 16)
    parents = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    c, wts, y = torch.zeros(4, device="cuda"), torch.zeros(4, 2, device="cuda"), torch.zeros(8, 64, device="cuda")
    logits, out = torch.zeros(4, 16, device="cuda"), bs.outputs(2)
    calls = [lambda **k: bs.select(logits, c, out=out, **k), lambda **k: reorder_states(x, parents, **k),
             lambda **k: lin(x, out=logits, **k), lambda **k: moe.group_rows(ids, 3, out=groups, **k),
             lambda **k: moe.grouped_product(x, w, groups, out=y, **k),
             lambda **k: moe.combine(y, groups, wts, out=torch.zeros(4, 64, device="cuda"), **k),
             lambda **k: layer(x, ids, wts, out=torch.zeros_like(x), **k)]

    class Elsewhere:
        device_index, cuda_stream = 1, 0

    other = new_stream()
    for call in calls:
        call()
        call(stream=other)
        with pytest.raises(ValueError, match="the stream on cuda:1"):
            call(stream=Elsewhere())
    torch.cuda.synchronize()
    monkeypatch.setattr(beam, "_current_device", lambda: 1)
    for call in calls + [lambda: W4Linear(q, s)]:
        with pytest.raises(ValueError, match="the stream on cuda:1"):
            call()

"""Checks that the Python front ends of the beam, 4-bit and expert calls make
before anything reaches a device, on CPU tensors."""
import pytest
import torch

from hi_amd.beam import BeamSearch


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

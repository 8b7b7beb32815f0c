"""SpecVerifier takes its tensors in the documented shapes alone: one with as many
values in another order would be read wrongly.  (Checked before the tensors'
device, so without a GPU.)"""
import pytest
import torch

from hi_amd.speculative import SpecVerifier

B, K, V = 4, 2, 10
I, F = torch.int32, torch.float32


def call(**changed):
    verifier = SpecVerifier(B, K, V, device="cpu")
    args = dict(target_probs=torch.zeros(B, K + 1, V), draft_tokens=torch.zeros(B, K, dtype=I),
                uniforms=torch.zeros(B, K + 1), draft_probs=torch.zeros(B, K, V), draft_len=torch.zeros(B, dtype=I),
                out={"tokens": torch.zeros(B, K + 1, dtype=I), "counts": torch.zeros(B, dtype=I)})
    out = {k: changed.pop(k) for k in ("tokens", "counts") if k in changed}
    args["out"].update(out)
    args.update(changed)
    verifier(**args)


@pytest.mark.parametrize("name,shapes,dtype", [
    ("draft_tokens", [(K, B), (B * K,), (B, K, 1), (1, B * K)], I), ("uniforms", [(K + 1, B), (B * (K + 1),)], F),
    ("tokens", [(K + 1, B), (B * (K + 1),), (1, B, K + 1)], I), ("counts", [(B, 1), (1, B), (2, 2)], I),
    ("draft_len", [(B, 1), (1, B), (2, 2)], I)])
def test_other_shapes_are_refused(name, shapes, dtype):
    for shape in shapes:
        with pytest.raises(ValueError, match=name.replace("counts", "out counts") + " must be"):
            call(**{name: torch.zeros(shape, dtype=dtype)})


def test_documented_shapes_go_on_to_the_device():
    with pytest.raises(ValueError, match="CUDA"):
        call()
    with pytest.raises(ValueError, match="CUDA"):
        call(draft_len=None, draft_probs=None)
    with pytest.raises(ValueError, match="contiguous"):
        call(uniforms=torch.zeros(K + 1, B).t())


def test_no_drafts():
    verifier = SpecVerifier(B, 0, V, device="cpu")
    with pytest.raises(ValueError, match="CUDA"):
        verifier(torch.zeros(B, 1, V), torch.zeros(B, 0, dtype=I), torch.zeros(B, 1))

"""Speculative decoding: verification of sampled drafts against the target's
probabilities (``hi_rocm_spec_verify_sampled``)."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ._lib import check, load
from .beam import _CODES, _on, _ptr, _stream, _zeroed

_INT, _FLOAT = torch.int32, torch.float32


def _shaped(what: str, name: str, t: torch.Tensor, dtype: torch.dtype, *shape: int) -> None:
    # (by shape, not by number: [drafts][batch] has as many values as [batch][drafts])
    if t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous {dtype} {''.join(f'[{n}]' for n in shape)} tensor")


class SpecVerifier:
    """The rejection rule for up to ``max_batch`` requests of ``max_draft``
    drafts over ``vocab`` tokens, with its own workspace (one stream at a
    time), which is allocated and zeroed on ``stream`` and ready for any when
    this returns."""

    def __init__(self, max_batch: int, max_draft: int, vocab: int, device="cuda",
                 stream: Optional[torch.cuda.Stream] = None):
        if max_draft < 0:
            raise ValueError(f"spec verifier: {max_draft} drafts")
        self.max_batch, self.max_draft, self.vocab = max_batch, max_draft, vocab
        nbytes = ctypes.c_size_t()
        check(load().hi_rocm_spec_sampled_workspace_bytes(max_batch, vocab, ctypes.byref(nbytes)))
        self._bytes = nbytes.value
        self.workspace = _zeroed(nbytes.value, device, stream)
        self._device, self._verify = self.workspace.get_device(), load().hi_rocm_spec_verify_sampled

    def outputs(self, batch: int, stream: Optional[torch.cuda.Stream] = None) -> dict:
        """Output tensors of a call for ``batch`` requests."""
        dev = self.workspace.device

        def make():
            return {"tokens": torch.empty(batch, self.max_draft + 1, dtype=torch.int32, device=dev),
                    "counts": torch.empty(batch, dtype=torch.int32, device=dev)}
        if stream is None:
            return make()
        with torch.cuda.stream(stream):
            return make()

    def __call__(self, target_probs: torch.Tensor, draft_tokens: torch.Tensor, uniforms: torch.Tensor,
                 draft_probs: Optional[torch.Tensor] = None, draft_len: Optional[torch.Tensor] = None,
                 out: Optional[dict] = None, stream: Optional[torch.cuda.Stream] = None) -> dict:
        """``target_probs`` float32 or bfloat16 [batch][max_draft + 1][vocab]
        (row i after a request's first i drafts), ``draft_tokens`` int32
        [batch][max_draft], ``uniforms`` float32 [batch][max_draft + 1] in [0,
        1): number i for draft i, the last for the token drawn behind the
        accepted ones.  ``draft_probs`` as target_probs, [batch][max_draft]
        [vocab], or None for drafts that were not sampled; ``draft_len`` int32
        [batch].  Returns ``tokens`` int32 [batch][max_draft + 1] (accepted
        drafts, drawn token, then -1) and ``counts`` int32 [batch]."""
        # (each check is written out: a call takes longer on the host than its kernel)
        what = "spec verifier"
        K, V, p, q, dev = self.max_draft, self.vocab, target_probs, draft_probs, self._device
        code = _CODES.get(p.dtype)
        if code is None or p.dim() != 3 or p.size(1) != K + 1 or p.size(2) != V or (V > 1 and p.stride(2) != 1):
            raise ValueError(f"{what}: target_probs must be a float32 or bfloat16 [batch][{K + 1}][{V}] tensor, values "
                             "contiguous")
        batch = p.size(0)
        if not 0 < batch <= self.max_batch:
            raise ValueError(f"{what}: {batch} requests, at most {self.max_batch}")
        q_at = q_batch = q_row = 0
        if q is not None:
            if q.dtype is not p.dtype or q.dim() != 3 or q.size(0) != batch or q.size(1) != K or q.size(2) != V or (
                    V > 1 and K > 0 and q.stride(2) != 1):
                raise ValueError(f"{what}: draft_probs must be a {p.dtype} [{batch}][{K}][{V}] tensor, values contiguous")
            q_at, q_batch, q_row = q.data_ptr(), q.stride(0), q.stride(1)
        if out is None:
            out = self.outputs(batch, stream)
        tokens, counts = out["tokens"], out["counts"]
        if not (draft_tokens.dtype is _INT and tokens.dtype is _INT and counts.dtype is _INT and
                uniforms.dtype is _FLOAT and draft_tokens.shape == (batch, K) and tokens.shape == (batch, K + 1) and
                counts.shape == (batch,) and uniforms.shape == (batch, K + 1) and draft_tokens.is_contiguous() and
                tokens.is_contiguous() and counts.is_contiguous() and uniforms.is_contiguous()):
            _shaped(what, "draft_tokens", draft_tokens, _INT, batch, K)
            _shaped(what, "uniforms", uniforms, _FLOAT, batch, K + 1)
            _shaped(what, "out tokens", tokens, _INT, batch, K + 1)
            _shaped(what, "out counts", counts, _INT, batch)
        if draft_len is not None:
            _shaped(what, "draft_len", draft_len, _INT, batch)
        if not (p.get_device() == draft_tokens.get_device() == uniforms.get_device() == tokens.get_device() ==
                counts.get_device() == dev) or dev < 0 or q is not None or draft_len is not None:
            _on(what, dev, p, draft_tokens, uniforms, q, draft_len, tokens, counts)
        status = self._verify(
            p.data_ptr(), code, batch, K, V, p.stride(0), p.stride(1), q_at, q_batch, q_row, draft_tokens.data_ptr(),
            _ptr(draft_len), uniforms.data_ptr(), tokens.data_ptr(), counts.data_ptr(), self.workspace.data_ptr(),
            self._bytes, _stream(what, dev, stream))
        if status:
            check(status)
        return out


__all__ = ["SpecVerifier"]

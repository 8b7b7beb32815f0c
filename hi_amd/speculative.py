"""Speculative decoding: verification of sampled drafts against the target's
probabilities (``hi_rocm_spec_verify_sampled``)."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ._lib import check, load
from .beam import _CODES, _F32, _I32, _on, _ptr, _stream, _vector


class SpecVerifier:
    """The rejection rule for up to ``max_batch`` requests of ``max_draft``
    drafts over ``vocab`` tokens, with its own workspace (one stream at a
    time)."""

    def __init__(self, max_batch: int, max_draft: int, vocab: int, device="cuda"):
        if max_draft < 0:
            raise ValueError(f"spec verifier: {max_draft} drafts")
        self.max_batch, self.max_draft, self.vocab = max_batch, max_draft, vocab
        nbytes = ctypes.c_size_t()
        check(load().hi_rocm_spec_sampled_workspace_bytes(max_batch, vocab, ctypes.byref(nbytes)))
        self._bytes = nbytes.value
        self.workspace = torch.zeros(nbytes.value, dtype=torch.uint8, device=device)

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
        what = "spec verifier"
        K, V = self.max_draft, self.vocab
        code = _CODES.get(target_probs.dtype)
        if code is None or target_probs.dim() != 3 or target_probs.shape[1:] != (K + 1, V) or (
                V > 1 and target_probs.stride(2) != 1):
            raise ValueError(f"{what}: target_probs must be a float32 or bfloat16 [batch][{K + 1}][{V}] tensor, values "
                             "contiguous")
        batch = target_probs.size(0)
        if not 0 < batch <= self.max_batch:
            raise ValueError(f"{what}: {batch} requests, at most {self.max_batch}")
        strides = (0, 0)
        if draft_probs is not None:
            if draft_probs.dtype != target_probs.dtype or draft_probs.shape != (batch, K, V) or (
                    V > 1 and K > 0 and draft_probs.stride(2) != 1):
                raise ValueError(f"{what}: draft_probs must be a {target_probs.dtype} [{batch}][{K}][{V}] tensor, values "
                                 "contiguous")
            strides = draft_probs.stride(0), draft_probs.stride(1)
        _vector(what, "draft_tokens", draft_tokens, _I32, batch * K)
        _vector(what, "uniforms", uniforms, _F32, batch * (K + 1))
        if draft_len is not None:
            _vector(what, "draft_len", draft_len, _I32, batch)
        if out is None:
            out = self.outputs(batch, stream)
        tokens, counts = out["tokens"], out["counts"]
        _vector(what, "out tokens", tokens, _I32, batch * (K + 1))
        _vector(what, "out counts", counts, _I32, batch)
        workspace = self.workspace
        dev = workspace.get_device()
        _on(what, dev, target_probs, draft_tokens, uniforms, draft_probs, draft_len, tokens, counts)
        check(load().hi_rocm_spec_verify_sampled(
            target_probs.data_ptr(), code, batch, K, V, target_probs.stride(0), target_probs.stride(1),
            _ptr(draft_probs), strides[0], strides[1], draft_tokens.data_ptr(), _ptr(draft_len), uniforms.data_ptr(),
            tokens.data_ptr(), counts.data_ptr(), workspace.data_ptr(), self._bytes, _stream(what, dev, stream)))
        return out


__all__ = ["SpecVerifier"]

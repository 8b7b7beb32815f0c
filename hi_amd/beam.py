"""Beam search: the selection over a request's beams and the vocabulary, and
the reordering of the beams' states (``hi_rocm_beam_select``,
``hi_rocm_beam_reorder``).

Everything stays on the device; calls only enqueue kernels, on the current
stream or the one given, and may be captured in a graph.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from ._lib import check, load
from .sampler import _stream_ptr


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _empty(shape, dtype, device, stream: Optional[torch.cuda.Stream]) -> torch.Tensor:
    """A new output, of the stream that writes it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _same_device(what: str, dev: torch.device, **tensors) -> None:
    if dev.type != "cuda":
        raise ValueError(f"{what}: needs CUDA tensors")
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: {name} is on {t.device}, not on {dev}")


def _vector(what: str, name: str, t: torch.Tensor, dtypes, numel: int) -> None:
    if t.dtype not in dtypes or not t.is_contiguous() or t.numel() != numel:
        raise ValueError(f"{what}: {name} must be a contiguous {' or '.join(str(d) for d in dtypes)} tensor of "
                         f"{numel} values")


class BeamSearch:
    """Selection for up to ``max_batch`` requests of ``beams`` beams over
    ``vocab`` tokens, ``n_out`` candidates each, with its own workspace (one
    stream at a time)."""

    def __init__(self, max_batch: int, beams: int, vocab: int, n_out: Optional[int] = None, device="cuda"):
        self.max_batch, self.beams, self.vocab = max_batch, beams, vocab
        self.n_out = beams if n_out is None else n_out
        nbytes = ctypes.c_size_t()
        check(load().hi_rocm_beam_workspace_bytes(max_batch, beams, vocab, self.n_out, ctypes.byref(nbytes)))
        self.workspace = torch.empty(nbytes.value, dtype=torch.uint8, device=device)

    def outputs(self, batch: int, stream: Optional[torch.cuda.Stream] = None) -> dict:
        """Output tensors of ``select`` for ``batch`` requests."""
        def new(dtype):
            return _empty((batch, self.n_out), dtype, self.workspace.device, stream)

        return {"scores": new(torch.float32), "tokens": new(torch.int32), "parents": new(torch.int32),
                "finished": new(torch.uint8)}

    def select(self, logits: torch.Tensor, scores: torch.Tensor, finished: Optional[torch.Tensor] = None,
               eos_id: Optional[int] = None, mask_words: Optional[torch.Tensor] = None,
               out: Optional[dict] = None, stream: Optional[torch.cuda.Stream] = None) -> dict:
        """The first ``n_out`` candidates of each request: ``scores``,
        ``tokens``, ``parents`` (beam within the request) and ``finished``,
        [batch][n_out] each.  ``logits`` [batch * beams][vocab] f32 or bf16;
        ``scores`` f32 and ``finished`` uint8 or bool of batch * beams values;
        ``mask_words`` int32 [batch * beams][ceil(vocab / 32)]."""
        what = "beam select"
        if logits.dim() != 2 or logits.shape[1] != self.vocab or logits.stride(1) != 1:
            raise ValueError(f"{what}: logits must be [batch * beams][{self.vocab}], tokens contiguous")
        if logits.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"{what}: logits must be float32 or bfloat16")
        rows = logits.shape[0]
        batch = rows // self.beams
        if rows != batch * self.beams or not 0 < batch <= self.max_batch:
            raise ValueError(f"{what}: {rows} rows for {self.beams} beams, at most {self.max_batch} requests")
        _vector(what, "scores", scores, (torch.float32,), rows)
        if finished is not None:
            _vector(what, "finished", finished, (torch.uint8, torch.bool), rows)
            if eos_id is None:
                raise ValueError(f"{what}: finished beams need an eos_id")
        if mask_words is not None:
            _vector(what, "mask_words", mask_words, (torch.int32,), rows * ((self.vocab + 31) // 32))
        if eos_id is not None and not 0 <= eos_id < self.vocab:
            raise ValueError(f"{what}: eos_id outside the vocabulary")
        if out is None:
            out = self.outputs(batch, stream)
        n = batch * self.n_out
        _vector(what, "out scores", out["scores"], (torch.float32,), n)
        _vector(what, "out tokens", out["tokens"], (torch.int32,), n)
        _vector(what, "out parents", out["parents"], (torch.int32,), n)
        _vector(what, "out finished", out["finished"], (torch.uint8, torch.bool), n)
        _same_device(what, self.workspace.device, logits=logits, scores=scores, finished=finished,
                     mask_words=mask_words, **{f"out {k}": v for k, v in out.items()})
        check(load().hi_rocm_beam_select(
            logits.data_ptr(), _lib.DTYPE_F32 if logits.dtype == torch.float32 else _lib.DTYPE_BF16, batch, self.beams,
            self.vocab, max(logits.stride(0), self.vocab), scores.data_ptr(), _ptr(finished),
            _lib.BEAM_NO_EOS if eos_id is None else eos_id, _ptr(mask_words), self.n_out, out["scores"].data_ptr(),
            out["tokens"].data_ptr(), out["parents"].data_ptr(), out["finished"].data_ptr(),
            self.workspace.data_ptr(), self.workspace.numel(), _stream_ptr(stream)))
        return out


def _one_stride(t: torch.Tensor, dims) -> tuple:
    """(count, stride in elements) of consecutive dims that step evenly."""
    dims = [d for d in dims if t.shape[d] != 1]
    if not dims:
        return 1, 0
    for a, b in zip(dims, dims[1:]):
        if t.stride(a) != t.shape[b] * t.stride(b):
            raise ValueError("reorder states: dimensions of the state do not step evenly")
    n = 1
    for d in dims:
        n *= t.shape[d]
    return n, t.stride(dims[-1])


def reorder_states(src: torch.Tensor, parents: torch.Tensor, dst: Optional[torch.Tensor] = None, row_dim: int = 0,
                   length_dim: Optional[int] = None, lengths: Optional[torch.Tensor] = None,
                   stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Row b * beams + j of ``dst`` (along ``row_dim``) becomes row b * beams +
    parents[b][j] of ``src``.  ``parents``: int32 [batch][beams].  Without
    ``dst`` the rows move in place.  With ``lengths`` (int32 [batch]) only the
    first lengths[b] positions along ``length_dim`` (behind ``row_dim``, what
    follows it contiguous) move.  Returns the reordered state."""
    what = "reorder states"
    if dst is None:
        dst = src
    if parents.dim() != 2 or parents.dtype != torch.int32 or not parents.is_contiguous():
        raise ValueError(f"{what}: parents must be a contiguous int32 [batch][beams] tensor")
    batch, beams = parents.shape
    nd = src.dim()
    if not 0 <= row_dim < nd or src.shape[row_dim] != batch * beams:
        raise ValueError(f"{what}: dimension {row_dim} must have batch * beams = {batch * beams} rows")
    if src.numel() == 0:
        raise ValueError(f"{what}: an empty state")
    if dst.shape != src.shape or dst.stride() != src.stride() or dst.dtype != src.dtype:
        raise ValueError(f"{what}: dst must have the shape, strides and type of src")
    if (lengths is None) != (length_dim is None):
        raise ValueError(f"{what}: lengths and length_dim go together")
    if lengths is not None:
        if not row_dim < length_dim < nd:
            raise ValueError(f"{what}: length_dim must follow row_dim")
        _vector(what, "lengths", lengths, (torch.int32,), batch)
    es = src.element_size()
    # the trailing dimensions that are contiguous: positions of a length, or
    # one position of everything
    inner = 1
    first = nd
    stop = length_dim + 1 if length_dim is not None else row_dim + 1
    while first > stop and (src.shape[first - 1] == 1 or src.stride(first - 1) == inner):
        first -= 1
        inner *= src.shape[first]
    if length_dim is not None:
        if first != stop or (src.shape[length_dim] != 1 and src.stride(length_dim) != inner):
            raise ValueError(f"{what}: what lies behind length_dim, and its positions, must be contiguous")
        positions, mids = src.shape[length_dim], range(row_dim + 1, length_dim)
    else:
        positions, mids = 1, range(row_dim + 1, first)
    outer, outer_stride = _one_stride(src, range(row_dim))
    mid, mid_stride = _one_stride(src, mids)
    _same_device(what, src.device, parents=parents, dst=dst, lengths=lengths)
    check(load().hi_rocm_beam_reorder(
        src.data_ptr(), dst.data_ptr(), parents.data_ptr(), batch, beams, outer, outer_stride * es,
        src.stride(row_dim) * es, mid, mid_stride * es, positions, inner * es, _ptr(lengths), _stream_ptr(stream)))
    return dst


__all__ = ["BeamSearch", "reorder_states"]

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


_CODES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


# The checks below run before every call, next to kernels of a few
# microseconds: torch.cuda.current_stream() alone takes 2.7 us, comparing two
# torch.device objects more than their indexes.

def _stream(what: str, dev: int, stream: Optional[torch.cuda.Stream]) -> int:
    """The handle of ``stream``, or of the current device's current one, which
    must be on CUDA device ``dev`` as the tensors are."""
    at = _current_device() if stream is None else stream.device_index
    if at != dev:
        raise ValueError(f"{what}: tensors on cuda:{dev}, the stream on cuda:{at}")
    return _raw_stream(dev) if stream is None else stream.cuda_stream


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _empty(shape, dtype, device, stream: Optional[torch.cuda.Stream]) -> torch.Tensor:
    """A new output, of the stream that writes it."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _zeroed(nbytes: int, device, stream: Optional[torch.cuda.Stream]) -> torch.Tensor:
    """A workspace whose bytes are 0, of ``stream``.  The fill has ended when this
    returns, as a first call on another stream would not wait for it (in a
    capture it is the graph's, whose calls come after it)."""
    if stream is None:
        made = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        if made.get_device() >= 0:
            stream = torch.cuda.current_stream(made.get_device())
    else:
        with torch.cuda.stream(stream):
            made = torch.zeros(nbytes, dtype=torch.uint8, device=device)
        if made.get_device() != stream.device_index:
            raise ValueError(f"a workspace on {made.device}, its stream on cuda:{stream.device_index}")
    if stream is not None:
        with torch.cuda.stream(stream):
            capturing = torch.cuda.is_current_stream_capturing()
        if not capturing:
            stream.synchronize()
    return made


def _on(what: str, dev: int, *tensors: Optional[torch.Tensor]) -> None:
    """All tensors on CUDA device ``dev``."""
    if dev < 0:
        raise ValueError(f"{what}: needs CUDA tensors")
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{what}: a tensor on {t.device}, not on cuda:{dev}")


def _vector(what: str, name: str, t: torch.Tensor, dtypes, numel: int) -> None:
    if t.dtype not in dtypes or t.numel() != numel or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be a contiguous {' or '.join(str(d) for d in dtypes)} tensor of "
                         f"{numel} values")


_F32, _I32, _FLAG = (torch.float32,), (torch.int32,), (torch.uint8, torch.bool)


class BeamSearch:
    """Selection for up to ``max_batch`` requests of ``beams`` beams over
    ``vocab`` tokens, ``n_out`` candidates each, with its own workspace (one
    stream at a time), of ``stream``."""

    def __init__(self, max_batch: int, beams: int, vocab: int, n_out: Optional[int] = None, device="cuda",
                 stream: Optional[torch.cuda.Stream] = None):
        self.max_batch, self.beams, self.vocab = max_batch, beams, vocab
        self.n_out = beams if n_out is None else n_out
        nbytes = ctypes.c_size_t()
        check(load().hi_rocm_beam_workspace_bytes(max_batch, beams, vocab, self.n_out, ctypes.byref(nbytes)))
        self._bytes = nbytes.value
        self.workspace = _empty((nbytes.value,), torch.uint8, device, stream)

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
        [batch][n_out] each.  ``logits`` [batch * beams][vocab] f32 or bf16, rows at
        least vocab apart (no expanded row);
        ``scores`` f32 and ``finished`` uint8 or bool of batch * beams values;
        ``mask_words`` int32 [batch * beams][ceil(vocab / 32)]."""
        what = "beam select"
        K, V = self.beams, self.vocab
        if logits.dim() != 2 or logits.size(1) != V or logits.stride(1) != 1:
            raise ValueError(f"{what}: logits must be [batch * beams][{V}], tokens contiguous")
        dtype = _CODES.get(logits.dtype)
        if dtype is None:
            raise ValueError(f"{what}: logits must be float32 or bfloat16")
        rows = logits.size(0)
        batch = rows // K
        if rows != batch * K or not 0 < batch <= self.max_batch:
            raise ValueError(f"{what}: {rows} rows for {K} beams, at most {self.max_batch} requests")
        stride = logits.stride(0) if rows > 1 else V  # (a single row's says nothing)
        if stride < V:
            raise ValueError(f"{what}: rows of logits overlap")
        _vector(what, "scores", scores, _F32, rows)
        if finished is not None:
            _vector(what, "finished", finished, _FLAG, rows)
            if eos_id is None:
                raise ValueError(f"{what}: finished beams need an eos_id")
        if mask_words is not None:
            _vector(what, "mask_words", mask_words, _I32, rows * ((V + 31) // 32))
        if eos_id is not None and not 0 <= eos_id < V:
            raise ValueError(f"{what}: eos_id outside the vocabulary")
        if out is None:
            out = self.outputs(batch, stream)
        n = batch * self.n_out
        o_scores, o_tokens, o_parents, o_finished = out["scores"], out["tokens"], out["parents"], out["finished"]
        _vector(what, "out scores", o_scores, _F32, n)
        _vector(what, "out tokens", o_tokens, _I32, n)
        _vector(what, "out parents", o_parents, _I32, n)
        _vector(what, "out finished", o_finished, _FLAG, n)
        if self.n_out != K and (o_scores.data_ptr() == scores.data_ptr() or
                                (finished is not None and o_finished.data_ptr() == finished.data_ptr())):
            raise ValueError(f"{what}: outputs over inputs need n_out = beams")
        ws = self.workspace
        _on(what, ws.get_device(), logits, scores, finished, mask_words, o_scores, o_tokens, o_parents, o_finished)
        check(load().hi_rocm_beam_select(
            logits.data_ptr(), dtype, batch, K, V, stride, scores.data_ptr(), _ptr(finished),
            _lib.BEAM_NO_EOS if eos_id is None else eos_id, _ptr(mask_words), self.n_out, o_scores.data_ptr(),
            o_tokens.data_ptr(), o_parents.data_ptr(), o_finished.data_ptr(), ws.data_ptr(), self._bytes,
            _stream(what, ws.get_device(), stream)))
        return out


def _one_stride(shape, strides, a: int, b: int) -> tuple:
    """(count, stride in elements) of dimensions [a, b), which step evenly."""
    n, step = 1, 0
    for d in range(b - 1, a - 1, -1):
        if shape[d] != 1:
            if n != 1 and strides[d] != n * step:
                raise ValueError("reorder states: dimensions of the state do not step evenly")
            step = step if n != 1 else strides[d]
            n *= shape[d]
    return n, step


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
    if parents.dim() != 2 or parents.dtype is not torch.int32 or not parents.is_contiguous():
        raise ValueError(f"{what}: parents must be a contiguous int32 [batch][beams] tensor")
    batch, beams = parents.shape
    shape, strides = src.shape, src.stride()
    nd = len(shape)
    if not 0 <= row_dim < nd or shape[row_dim] != batch * beams:
        raise ValueError(f"{what}: dimension {row_dim} must have batch * beams = {batch * beams} rows")
    if src.numel() == 0:
        raise ValueError(f"{what}: an empty state")
    if dst is not src and (dst.shape != shape or dst.stride() != strides or dst.dtype is not src.dtype):
        raise ValueError(f"{what}: dst must have the shape, strides and type of src")
    if (lengths is None) != (length_dim is None):
        raise ValueError(f"{what}: lengths and length_dim go together")
    if lengths is not None:
        if not row_dim < length_dim < nd:
            raise ValueError(f"{what}: length_dim must follow row_dim")
        _vector(what, "lengths", lengths, _I32, batch)
    es = src.element_size()
    # the trailing dimensions that are contiguous: what lies behind a length,
    # or one position of everything
    inner, first = 1, nd
    stop = row_dim + 1 if length_dim is None else length_dim + 1
    while first > stop and (shape[first - 1] == 1 or strides[first - 1] == inner):
        first -= 1
        inner *= shape[first]
    if length_dim is None:
        positions, mid_end = 1, first
    else:
        if first != stop or (shape[length_dim] != 1 and strides[length_dim] != inner):
            raise ValueError(f"{what}: what lies behind length_dim, and its positions, must be contiguous")
        positions, mid_end = shape[length_dim], length_dim
    outer, outer_stride = _one_stride(shape, strides, 0, row_dim)
    mid, mid_stride = _one_stride(shape, strides, row_dim + 1, mid_end)
    _on(what, src.get_device(), parents, dst, lengths)
    check(load().hi_rocm_beam_reorder(
        src.data_ptr(), dst.data_ptr(), parents.data_ptr(), batch, beams, outer, outer_stride * es,
        strides[row_dim] * es, mid, mid_stride * es, positions, inner * es, _ptr(lengths),
        _stream(what, src.get_device(), stream)))
    return dst


__all__ = ["BeamSearch", "reorder_states"]

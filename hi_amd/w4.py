"""Products with 4-bit weights and group scales (``hi_rocm_w4_pack``,
``hi_rocm_w4_linear``): projections and output heads of quantised models for
the rows of a decode step."""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from ._lib import check, load
from .beam import _CODES, _empty, _on, _ptr, _stream


def quantize_w4(weight: torch.Tensor, group: int = 32, symmetric: bool = True, scale_dtype=torch.bfloat16):
    """Rounds a weight [n][k] to 4 bits: (q, scales, zeros) for ``W4Linear``,
    zeros None when symmetric.  Scales are rounded to their type first, so the
    nearest of the 16 values is taken for what will be multiplied."""
    n, k = weight.shape
    if k % group != 0:
        raise ValueError(f"quantize_w4: {k} inputs are no multiple of the group of {group}")
    w = weight.float().view(n, k // group, group)
    if symmetric:
        scale = (w.abs().amax(2) / 7.0).to(scale_dtype)
        zero, z = None, 8.0
    else:
        lo, hi = w.amin(2).clamp_(max=0.0), w.amax(2).clamp_(min=0.0)
        scale = ((hi - lo) / 15.0).to(scale_dtype)
    s = scale.float()
    s = torch.where(s > 0, s, torch.ones_like(s))
    if not symmetric:
        zero = torch.round(-lo / s).clamp_(0.0, 15.0).to(scale_dtype)
        z = zero.float()[:, :, None]
    q = torch.round(w / s[:, :, None] + z).clamp_(0.0, 15.0).to(torch.uint8).view(n, k)
    return q[:, 0::2] | (q[:, 1::2] << 4), scale, zero


class W4Linear:
    """y = x w^T + bias for the 4-bit weight w = (q - zero) * scale, laid out
    once.  ``q`` uint8 [n][k / 2] (input 2 j in byte j's low nibble),
    ``scales`` and ``zeros`` (None: 8) [n][k / group] float32 or bfloat16,
    group 32, 64 or 128; ``bias`` float32 [n] or None.  They are packed on
    ``stream``, which must come after what made them, and need not be kept."""

    def __init__(self, q: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None,
                 bias: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None):
        what = "w4 linear"
        if q.dim() != 2 or q.dtype != torch.uint8 or not q.is_contiguous():
            raise ValueError(f"{what}: q must be a contiguous uint8 [n][k / 2] tensor")
        self.n, self.k = q.shape[0], q.shape[1] * 2
        if (scales.dim() != 2 or scales.shape[0] != self.n or scales.shape[1] == 0 or
                self.k % scales.shape[1] != 0 or scales.dtype not in _CODES or not scales.is_contiguous()):
            raise ValueError(f"{what}: scales must be a contiguous float32 or bfloat16 [n][k / group] tensor")
        self.group = self.k // scales.shape[1]
        if zeros is not None and (zeros.shape != scales.shape or zeros.dtype != scales.dtype or
                                  not zeros.is_contiguous()):
            raise ValueError(f"{what}: zeros must be like scales")
        if bias is not None and (bias.shape != (self.n,) or bias.dtype != torch.float32 or not bias.is_contiguous()):
            raise ValueError(f"{what}: bias must be a contiguous float32 [n] tensor")
        _on(what, q.get_device(), scales, zeros, bias)
        self.bias, self.scale_dtype, self.has_zeros = bias, _CODES[scales.dtype], int(zeros is not None)
        lib, nbytes = load(), ctypes.c_size_t()
        check(lib.hi_rocm_w4_packed_bytes(self.n, self.k, self.group, self.scale_dtype, self.has_zeros,
                                          ctypes.byref(nbytes)))
        self._bytes = nbytes.value
        self.packed = _empty((nbytes.value,), torch.uint8, q.device, stream)
        check(lib.hi_rocm_w4_pack(q.data_ptr(), scales.data_ptr(), _ptr(zeros), self.scale_dtype, self.n, self.k,
                                  self.group, self.packed.data_ptr(), self.packed.numel(),
                                  _stream(what, q.get_device(), stream)))
        if stream is not None:  # (they may be freed before the packing has run)
            for t in (q, scales, zeros):
                if t is not None:
                    t.record_stream(stream)

    def __call__(self, x: torch.Tensor, out: Optional[torch.Tensor] = None, dtype=torch.float32,
                 stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """x bfloat16 [rows][k], rows starting on 16 bytes; returns out
        [rows][n] (a new tensor of ``dtype`` when not given)."""
        what = "w4 linear"
        n, k = self.n, self.k
        if x.dim() != 2 or x.dtype is not torch.bfloat16 or x.size(1) != k or x.stride(1) != 1 or x.size(0) == 0:
            raise ValueError(f"{what}: x must be a bfloat16 [rows][{k}] tensor, inputs contiguous")
        rows = x.size(0)
        if out is None:
            out = _empty((rows, n), dtype, x.device, stream)
        code = _CODES.get(out.dtype)
        if code is None or out.dim() != 2 or out.size(0) != rows or out.size(1) != n or out.stride(1) != 1:
            raise ValueError(f"{what}: out must be a float32 or bfloat16 [{rows}][{n}] tensor, outputs contiguous")
        packed = self.packed
        _on(what, packed.get_device(), x, out)
        # (a single row's stride says nothing)
        check(load().hi_rocm_w4_linear(
            x.data_ptr(), rows, x.stride(0) if rows > 1 else k, packed.data_ptr(), self._bytes, self.scale_dtype,
            self.has_zeros, n, k, self.group, _ptr(self.bias), out.data_ptr(), code,
            out.stride(0) if rows > 1 else n, _stream(what, packed.get_device(), stream)))
        return out


__all__ = ["W4Linear", "quantize_w4"]

"""Microscaled 4-bit floating point (MXFP4: blocks of 32 E2M1 codes with a
power-of-two scale): rounding, linear layers and expert layers whose products
take both operands in it (``hi_rocm_mx4_quantize``, ``hi_rocm_mx4_linear``,
``hi_rocm_mx4_grouped_product``)."""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from ._lib import DTYPE_BF16, DTYPE_MX4, check, load
from .beam import _CODES, _empty, _on, _ptr, _stream
from .moe import RowGroups

BLOCK = 32
_BYTE = torch.uint8


def _rows_of(what: str, name: str, x: torch.Tensor, k: Optional[int] = None) -> None:
    if x.dim() != 2 or x.dtype not in _CODES or x.numel() == 0 or x.stride(1) != 1 or (k and x.size(1) != k):
        raise ValueError(f"{what}: {name} must be a float32 or bfloat16 [rows][{k or 'k'}] tensor, values contiguous")
    if x.size(1) % BLOCK != 0:
        raise ValueError(f"{what}: {x.size(1)} values are no multiple of the block of {BLOCK}")


def _codes_of(what: str, codes: torch.Tensor, scales: torch.Tensor, dim: int) -> None:
    """codes [..][k / 2] and scales [..][k / 32], contiguous uint8."""
    if (codes.dim() != dim or codes.dtype != torch.uint8 or not codes.is_contiguous() or codes.numel() == 0 or
            codes.size(-1) % (BLOCK // 2) != 0):
        raise ValueError(f"{what}: codes must be a contiguous uint8 {'[experts]' * (dim - 2)}[rows][k / 2] tensor, k a "
                         f"multiple of {BLOCK}")
    if (scales.dtype != torch.uint8 or not scales.is_contiguous() or
            scales.shape != (*codes.shape[:-1], codes.size(-1) * 2 // BLOCK)):
        raise ValueError(f"{what}: scales must be a contiguous uint8 tensor of one byte for {BLOCK} values")


def _size(fn, *args) -> int:
    out = ctypes.c_size_t()
    check(fn(*args, ctypes.byref(out)))
    return out.value


def quantize_mx4(x: torch.Tensor, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                 stream: Optional[torch.cuda.Stream] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rounds x (float32 or bfloat16 [rows][k], rows on 16 bytes): codes uint8
    [rows][k / 2] (value 2 j in byte j's low nibble) and scales uint8 [rows]
    [k / 32], as ``Mx4Linear`` takes them."""
    # (checks written out where a call's host side takes longer than its kernel)
    what = "quantize mx4"
    code = _CODES.get(x.dtype)
    if code is None or x.dim() != 2 or x.numel() == 0 or x.stride(1) != 1 or x.size(1) % BLOCK != 0:
        _rows_of(what, "x", x)
    rows, k = x.size(0), x.size(1)
    if out is None:
        out = (_empty((rows, k // 2), _BYTE, x.device, stream), _empty((rows, k // BLOCK), _BYTE, x.device, stream))
    codes, scales = out
    if not (codes.dtype is _BYTE and scales.dtype is _BYTE and codes.dim() == 2 and scales.dim() == 2 and
            codes.size(0) == rows and codes.size(1) == k // 2 and scales.size(0) == rows and
            scales.size(1) == k // BLOCK and codes.is_contiguous() and scales.is_contiguous()):
        raise ValueError(f"{what}: out must be contiguous uint8 codes [{rows}][{k // 2}] and scales [{rows}][{k // BLOCK}]")
    dev = x.get_device()
    if dev < 0 or codes.get_device() != dev or scales.get_device() != dev:
        _on(what, dev, codes, scales)
    status = load().hi_rocm_mx4_quantize(x.data_ptr(), code, rows, k, x.stride(0) if rows > 1 else k, codes.data_ptr(),
                                         scales.data_ptr(), _stream(what, dev, stream))
    if status:
        check(status)
    return out


def dequantize_mx4(codes: torch.Tensor, scales: torch.Tensor, out: Optional[torch.Tensor] = None,
                   dtype=torch.bfloat16, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """The values [rows][k] of codes and scales, float32 or bfloat16 (``out``'s
    type)."""
    what = "dequantize mx4"
    if not (codes.dtype is _BYTE and scales.dtype is _BYTE and codes.dim() == 2 and scales.dim() == 2 and
            codes.numel() > 0 and codes.size(1) == scales.size(1) * (BLOCK // 2) and scales.size(0) == codes.size(0) and
            codes.is_contiguous() and scales.is_contiguous()):
        _codes_of(what, codes, scales, 2)
    rows, k = codes.size(0), codes.size(1) * 2
    if out is None:
        out = _empty((rows, k), dtype, codes.device, stream)
    code = _CODES.get(out.dtype)
    if code is None or out.dim() != 2 or out.size(0) != rows or out.size(1) != k or out.stride(1) != 1:
        raise ValueError(f"{what}: out must be a float32 or bfloat16 [{rows}][{k}] tensor, values contiguous")
    dev = codes.get_device()
    if dev < 0 or scales.get_device() != dev or out.get_device() != dev:
        _on(what, dev, scales, out)
    status = load().hi_rocm_mx4_dequantize(codes.data_ptr(), scales.data_ptr(), rows, k, out.data_ptr(), code,
                                           out.stride(0) if rows > 1 else k, _stream(what, dev, stream))
    if status:
        check(status)
    return out


class Mx4Rows:
    """Rows rounded once for several products: ``mx4_rows(x)``."""

    def __init__(self, rows: int, k: int, device="cuda", stream: Optional[torch.cuda.Stream] = None):
        self.rows, self.k = rows, k
        self._bytes = _size(load().hi_rocm_mx4_rows_bytes, rows, k)
        self.memory = _empty((self._bytes,), torch.uint8, device, stream)


def mx4_rows(x: torch.Tensor, out: Optional[Mx4Rows] = None, stream: Optional[torch.cuda.Stream] = None) -> Mx4Rows:
    """x (float32 or bfloat16 [rows][k], rows on 16 bytes) rounded, in the
    order that the products read."""
    what = "mx4 rows"
    _rows_of(what, "x", x)
    rows, k = x.shape
    if out is None:
        out = Mx4Rows(rows, k, device=x.device, stream=stream)
    if (out.rows, out.k) != (rows, k):
        raise ValueError(f"{what}: out is for {out.rows} rows of {out.k}")
    dev = x.get_device()
    _on(what, dev, out.memory)
    check(load().hi_rocm_mx4_rows(x.data_ptr(), _CODES[x.dtype], rows, k, x.stride(0) if rows > 1 else k,
                                  out.memory.data_ptr(), out._bytes, _stream(what, dev, stream)))
    return out


def _pack(what: str, codes: torch.Tensor, scales: torch.Tensor, experts: int, stream) -> torch.Tensor:
    """codes [..][n][k / 2] of ``experts`` weights in the products' layout."""
    dev, lib = codes.get_device(), load()
    _on(what, dev, scales)
    n, k = codes.size(-2), codes.size(-1) * 2
    nbytes = _size(lib.hi_rocm_mx4_packed_bytes, experts, n, k)
    packed = _empty((nbytes,), torch.uint8, codes.device, stream)
    check(lib.hi_rocm_mx4_pack(codes.data_ptr(), scales.data_ptr(), experts, n, k, packed.data_ptr(), nbytes,
                               _stream(what, dev, stream)))
    if stream is not None:  # (they may be freed before the packing has run)
        codes.record_stream(stream)
        scales.record_stream(stream)
    return packed


class Mx4Linear:
    """y = Q(x) w^T + bias for the weight w of ``codes`` uint8 [n][k / 2] and
    ``scales`` uint8 [n][k / 32] (``quantize_mx4``'s), laid out once; Q rounds x
    to the same format.  ``bias`` float32 [n] or None.  Codes and scales are
    packed on ``stream``, which must come after what made them, and need not be
    kept."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 stream: Optional[torch.cuda.Stream] = None):
        what = "mx4 linear"
        _codes_of(what, codes, scales, 2)
        self.n, self.k = codes.size(0), codes.size(1) * 2
        if bias is not None and (bias.shape != (self.n,) or bias.dtype != torch.float32 or not bias.is_contiguous()):
            raise ValueError(f"{what}: bias must be a contiguous float32 [n] tensor")
        _on(what, codes.get_device(), bias)
        self.bias = bias
        self.packed = _pack(what, codes, scales, 1, stream)
        self._bytes = self.packed.numel()
        self._device, self._linear = self.packed.get_device(), load().hi_rocm_mx4_linear
        self._work = {}  # rows: bytes of their workspace

    def __call__(self, x: Union[torch.Tensor, Mx4Rows], out: Optional[torch.Tensor] = None, dtype=torch.float32,
                 stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """x bfloat16 [rows][k], rows starting on 16 bytes, or ``mx4_rows`` of
        it; returns out [rows][n] (a new tensor of ``dtype`` when not given)."""
        what = "mx4 linear"
        n, k, dev, work, work_bytes = self.n, self.k, self._device, None, 0
        if isinstance(x, Mx4Rows):
            if x.k != k:
                raise ValueError(f"{what}: rows of {x.k}, the weight's are {k}")
            rows, at, code_x, stride, memory = x.rows, x.memory.data_ptr(), DTYPE_MX4, 0, x.memory
        else:
            if x.dim() != 2 or x.dtype is not torch.bfloat16 or x.size(1) != k or x.stride(1) != 1 or x.size(0) == 0:
                raise ValueError(f"{what}: x must be a bfloat16 [rows][{k}] tensor, inputs contiguous")
            rows, at, code_x, memory = x.size(0), x.data_ptr(), DTYPE_BF16, x
            stride = x.stride(0) if rows > 1 else k
        if out is None:
            out = _empty((rows, n), dtype, self.packed.device, stream)
        code = _CODES.get(out.dtype)
        if code is None or out.dim() != 2 or out.size(0) != rows or out.size(1) != n or (n > 1 and out.stride(1) != 1):
            raise ValueError(f"{what}: out must be a float32 or bfloat16 [{rows}][{n}] tensor, outputs contiguous")
        if memory.get_device() != dev or out.get_device() != dev:
            _on(what, dev, memory, out)
        if code_x == DTYPE_BF16:
            work_bytes = self._work.get(rows)
            if work_bytes is None:
                work_bytes = self._work[rows] = _size(load().hi_rocm_mx4_linear_workspace_bytes, rows, n, k)
            if work_bytes:  # a call's own: calls on several streams, or captured ones, share nothing
                work = _empty((work_bytes,), _BYTE, self.packed.device, stream)
        # (a single row's stride says nothing)
        status = self._linear(
            at, code_x, rows, stride, self.packed.data_ptr(), self._bytes, n, k, _ptr(self.bias), out.data_ptr(), code,
            out.stride(0) if rows > 1 else n, _ptr(work), work_bytes, _stream(what, dev, stream))
        if status:
            check(status)
        return out


class Mx4Experts:
    """``MoeExperts`` with 4-bit products: y[t] = sum_s w[t][s] down_e Q(silu(
    gate_e Q(x[t])) * (up_e Q(x[t]))), e = ids[t][s].  ``up`` uint8 [experts]
    [2 * inter][hidden / 2] (gate rows, then up rows) and ``down`` uint8
    [experts][hidden][inter / 2] with their scales; hidden and inter multiples
    of 32.  Activations go from f32 to 4 bits without a step between.  A
    token's terms are ``terms``, float32 or bfloat16, whatever the result's
    type, and their sum is f32.  float32 terms leave a bfloat16 result the one
    rounding at its end (0.0017 of its norm).  bfloat16 ones are rounded before
    they are weighted, each by up to 2^-8 of itself, which where a token's terms
    cancel is more than the result's own rounding (0.0024 of the norm for random
    ones), and halve what is written and read between the last two launches (8
    terms of 2048: 1,024 tokens 111 -> 101 us, 4,096 225 -> 185).  Weights are
    packed on ``stream`` and need not be kept; buffers for up to ``max_tokens``
    tokens are allocated once, of that stream too, and calls allocate nothing
    when ``out`` is given.  Calls on another stream must come after what was on
    ``stream`` when the layer was made, and end before the layer is dropped."""

    def __init__(self, up: torch.Tensor, up_scales: torch.Tensor, down: torch.Tensor, down_scales: torch.Tensor,
                 max_tokens: int, top_k: int, stream: Optional[torch.cuda.Stream] = None, terms=torch.float32):
        what = "mx4 experts"
        _codes_of(what, up, up_scales, 3)
        _codes_of(what, down, down_scales, 3)
        self.experts, self.hidden, self.inter = up.size(0), up.size(2) * 2, down.size(2) * 2
        if up.size(1) != 2 * self.inter or down.shape[:2] != (self.experts, self.hidden):
            raise ValueError(f"{what}: up [experts][2 * inter][hidden / 2] and down [experts][hidden][inter / 2]")
        if max_tokens <= 0 or top_k <= 0:
            raise ValueError(f"{what}: {max_tokens} tokens, top {top_k}")
        if terms not in _CODES:
            raise ValueError(f"{what}: terms must be float32 or bfloat16")
        _on(what, up.get_device(), down)
        self.max_tokens, self.top_k = max_tokens, top_k
        self._up = _pack(what, up, up_scales, self.experts, stream)
        self._down = _pack(what, down, down_scales, self.experts, stream)
        dev, lib, places = up.device, load(), max_tokens * top_k
        self._x_bytes = _size(lib.hi_rocm_mx4_rows_bytes, max_tokens, self.hidden)
        self._h_bytes = _size(lib.hi_rocm_mx4_rows_bytes, places, self.inter)
        # (of the stream that packed the weights: another's allocator may hand out memory
        # that its own work still uses, and take it back while this one's does)
        self._x = _empty((self._x_bytes,), _BYTE, dev, stream)
        self._h = _empty((self._h_bytes,), _BYTE, dev, stream)
        self._y = _empty((places, self.hidden), terms, dev, stream)
        self._groups = RowGroups(max_tokens, top_k, self.experts, device=dev, stream=stream)
        self._few = {}  # tokens: whether their rows need no rounding beforehand

    def __call__(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, out: Optional[torch.Tensor] = None,
                 stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """x bfloat16 [tokens][hidden], ids int32 and weights float32
        [tokens][top_k] from the router; returns [tokens][hidden] (bfloat16,
        or out's type).  The buffers serve one stream at a time."""
        what = "mx4 experts"
        k, E, H, I = self.top_k, self.experts, self.hidden, self.inter
        if x.dim() != 2 or x.dtype is not torch.bfloat16 or x.size(1) != H or x.stride(1) != 1:
            raise ValueError(f"{what}: x must be a bfloat16 [tokens][{H}] tensor, inputs contiguous")
        tokens = x.size(0)
        if not 0 < tokens <= self.max_tokens:
            raise ValueError(f"{what}: {tokens} tokens, at most {self.max_tokens}")
        if ids.shape != (tokens, k) or ids.dtype is not torch.int32 or not ids.is_contiguous():
            raise ValueError(f"{what}: ids must be a contiguous int32 [{tokens}][{k}] tensor")
        if weights.shape != (tokens, k) or weights.dtype is not torch.float32 or not weights.is_contiguous():
            raise ValueError(f"{what}: weights must be a contiguous float32 [{tokens}][{k}] tensor")
        if out is None:
            out = _empty((tokens, H), torch.bfloat16, x.device, stream)
        code = _CODES.get(out.dtype)
        if code is None or out.shape != (tokens, H) or out.stride(1) != 1:
            raise ValueError(f"{what}: out must be a float32 or bfloat16 [{tokens}][{H}] tensor")
        g, h, y = self._groups, self._h, self._y
        _on(what, h.get_device(), x, ids, weights, out)
        places, st, lib = tokens * k, _stream(what, h.get_device(), stream), load()
        order, slots, offsets = g.order.data_ptr(), g.slots.data_ptr(), g.offsets.data_ptr()
        at, code_x, stride = x.data_ptr(), DTYPE_BF16, x.stride(0) if tokens > 1 else H
        if self._few.get(tokens) is None:
            self._few[tokens] = _size(lib.hi_rocm_mx4_workspace_bytes, tokens, places, H) == 0
        if self._few[tokens]:  # the product rounds the rows as it reads them
            check(lib.hi_rocm_moe_group(ids.data_ptr(), tokens, k, E, order, slots, offsets, st))
        else:
            check(lib.hi_rocm_mx4_moe_prepare(ids.data_ptr(), tokens, k, E, order, slots, offsets, at, H, stride,
                                              self._x.data_ptr(), self._x_bytes, st))
            at, code_x = self._x.data_ptr(), DTYPE_MX4
        check(lib.hi_rocm_mx4_grouped_product(
            at, code_x, tokens, stride, order, k, offsets, places, E, self._up.data_ptr(), self._up.numel(), 2 * I, H, 1,
            h.data_ptr(), DTYPE_MX4, I, self._h_bytes, 0, 0, st))
        check(lib.hi_rocm_mx4_grouped_product(
            h.data_ptr(), DTYPE_MX4, places, 0, 0, 1, offsets, places, E, self._down.data_ptr(), self._down.numel(), H, I,
            0, y.data_ptr(), _CODES[y.dtype], H, 0, 0, 0, st))
        check(lib.hi_rocm_moe_combine(
            y.data_ptr(), _CODES[y.dtype], H, slots, offsets, E, weights.data_ptr(), tokens, k, H, out.data_ptr(), code,
            out.stride(0) if tokens > 1 else H, st))
        return out


__all__ = ["quantize_mx4", "dequantize_mx4", "Mx4Rows", "mx4_rows", "Mx4Linear", "Mx4Experts"]

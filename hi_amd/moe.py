"""The expert layer behind the MoE router: the router's pairs grouped by
expert, products over the groups, and the weighted sum of a token's experts
(``hi_rocm_moe_group``, ``hi_rocm_moe_grouped_product``,
``hi_rocm_moe_combine``)."""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import check, load
from .beam import _CODES, _empty, _on, _stream


class RowGroups:
    """The (token, slot) pairs p = token * top_k + slot sorted by expert:
    ``order`` (the pair in each place), ``slots`` (each pair's place) and
    ``offsets`` (expert e's places are offsets[e] .. offsets[e + 1])."""

    def __init__(self, tokens: int, top_k: int, experts: int, device="cuda",
                 stream: Optional[torch.cuda.Stream] = None):
        self.tokens, self.top_k, self.experts = tokens, top_k, experts
        self.order = _empty((tokens * top_k,), torch.int32, device, stream)
        self.slots = _empty((tokens * top_k,), torch.int32, device, stream)
        self.offsets = _empty((experts + 1,), torch.int32, device, stream)

    @property
    def places(self) -> int:
        return self.tokens * self.top_k


def group_rows(ids: torch.Tensor, experts: int, out: Optional[RowGroups] = None,
               stream: Optional[torch.cuda.Stream] = None) -> RowGroups:
    """Groups the router's ``ids`` (int32 [tokens][top_k]) by expert, stably.
    Pairs whose id names no expert come behind the groups."""
    what = "group rows"
    if ids.dim() != 2 or ids.dtype != torch.int32 or not ids.is_contiguous() or ids.numel() == 0:
        raise ValueError(f"{what}: ids must be a contiguous int32 [tokens][top_k] tensor")
    if out is None:
        out = RowGroups(ids.shape[0], ids.shape[1], experts, device=ids.device, stream=stream)
    if (out.tokens, out.top_k, out.experts) != (ids.shape[0], ids.shape[1], experts):
        raise ValueError(f"{what}: out is for {out.tokens} tokens, top {out.top_k} of {out.experts} experts")
    _on(what, ids.get_device(), out.order)
    check(load().hi_rocm_moe_group(ids.data_ptr(), out.tokens, out.top_k, experts, out.order.data_ptr(),
                                   out.slots.data_ptr(), out.offsets.data_ptr(),
                                   _stream(what, ids.get_device(), stream)))
    return out


def grouped_product(x: torch.Tensor, weight: torch.Tensor, groups: RowGroups, gather: bool = True,
                    swiglu: bool = False, out: Optional[torch.Tensor] = None, dtype=torch.bfloat16,
                    stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """out[i] = x[row(i)] weight[e]^T for place i of expert e; row(i) is the
    pair's token (``gather``) or i.  ``x`` bfloat16 [.][k], ``weight`` bfloat16
    [experts][cols][k]; with ``swiglu`` the columns are gate and up halves and
    out is silu(gate) * up, cols / 2 wide."""
    what = "grouped product"
    if weight.dim() != 3 or weight.dtype != torch.bfloat16 or not weight.is_contiguous():
        raise ValueError(f"{what}: weight must be a contiguous bfloat16 [experts][cols][k] tensor")
    experts, cols, k = weight.shape
    if experts != groups.experts:
        raise ValueError(f"{what}: weight has {experts} experts, the groups {groups.experts}")
    rows = groups.tokens if gather else groups.places
    if x.dim() != 2 or x.dtype != torch.bfloat16 or x.shape != (rows, k) or x.stride(1) != 1:
        raise ValueError(f"{what}: x must be a bfloat16 [{rows}][{k}] tensor, inputs contiguous")
    if swiglu and cols % 2:
        raise ValueError(f"{what}: gate and up columns: an even number")
    wide = cols // 2 if swiglu else cols
    if out is None:
        out = _empty((groups.places, wide), dtype, x.device, stream)
    if out.shape != (groups.places, wide) or out.dtype not in _CODES or out.stride(1) != 1:
        raise ValueError(f"{what}: out must be a float32 or bfloat16 [{groups.places}][{wide}] tensor")
    _on(what, x.get_device(), weight, groups.order, out)
    check(load().hi_rocm_moe_grouped_product(
        x.data_ptr(), rows, x.stride(0) if rows > 1 else k, groups.order.data_ptr() if gather else 0, groups.top_k,
        groups.offsets.data_ptr(), groups.places, experts, weight.data_ptr(), cols, k, int(swiglu), out.data_ptr(),
        _CODES[out.dtype], out.stride(0) if groups.places > 1 else wide, _stream(what, x.get_device(), stream)))
    return out


def combine(y: torch.Tensor, groups: RowGroups, weights: torch.Tensor, out: Optional[torch.Tensor] = None,
            dtype=torch.bfloat16, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """out[t] = sum_s weights[t][s] y[place of (t, s)], in slot order."""
    what = "combine"
    if y.dim() != 2 or y.shape[0] != groups.places or y.dtype not in _CODES or y.stride(1) != 1:
        raise ValueError(f"{what}: y must be a float32 or bfloat16 [{groups.places}][cols] tensor")
    if weights.shape != (groups.tokens, groups.top_k) or weights.dtype != torch.float32 or not weights.is_contiguous():
        raise ValueError(f"{what}: weights must be a contiguous float32 [tokens][top_k] tensor")
    if out is None:
        out = _empty((groups.tokens, y.shape[1]), dtype, y.device, stream)
    if out.shape != (groups.tokens, y.shape[1]) or out.dtype not in _CODES or out.stride(1) != 1:
        raise ValueError(f"{what}: out must be a float32 or bfloat16 [{groups.tokens}][{y.shape[1]}] tensor")
    _on(what, y.get_device(), groups.order, weights, out)
    check(load().hi_rocm_moe_combine(
        y.data_ptr(), _CODES[y.dtype], y.stride(0) if groups.places > 1 else y.shape[1], groups.slots.data_ptr(),
        groups.offsets.data_ptr(), groups.experts, weights.data_ptr(), groups.tokens, groups.top_k, y.shape[1],
        out.data_ptr(), _CODES[out.dtype], out.stride(0) if groups.tokens > 1 else y.shape[1],
        _stream(what, y.get_device(), stream)))
    return out


class MoeExperts:
    """The expert layer: y[t] = sum_s w[t][s] down_e (silu(gate_e x[t]) * (up_e
    x[t])), e = ids[t][s].  ``w_up`` bfloat16 [experts][2 * inter][hidden]
    (gate rows, then up rows), ``w_down`` bfloat16 [experts][hidden][inter].
    The activations between the two products are rounded to bfloat16, as in a
    bfloat16 model (a relative error of 0.0023 of a bfloat16 result, 0.0017
    with them in f32); all sums are f32.
    Buffers for up to ``max_tokens`` tokens are allocated once; calls allocate
    nothing when ``out`` is given."""

    def __init__(self, w_up: torch.Tensor, w_down: torch.Tensor, max_tokens: int, top_k: int):
        if (w_up.dim() != 3 or w_down.dim() != 3 or w_up.shape[1] % 2 or
                w_down.shape != (w_up.shape[0], w_up.shape[2], w_up.shape[1] // 2) or
                w_up.dtype is not torch.bfloat16 or w_down.dtype is not torch.bfloat16 or
                not w_up.is_contiguous() or not w_down.is_contiguous()):
            raise ValueError("moe experts: w_up [experts][2 * inter][hidden] and w_down [experts][hidden][inter], "
                             "contiguous bfloat16")
        _on("moe experts", w_up.get_device(), w_down)
        self.w_up, self.w_down, self.max_tokens, self.top_k = w_up, w_down, max_tokens, top_k
        self.experts, self.hidden, self.inter = w_up.shape[0], w_up.shape[2], w_down.shape[2]
        dev = w_up.device
        # The activations between the products are what the second product's
        # matrix instructions take, bf16; its results stay f32 until they are
        # summed.
        self._h = torch.empty(max_tokens * top_k, self.inter, dtype=torch.bfloat16, device=dev)
        self._y = torch.empty(max_tokens * top_k, self.hidden, dtype=torch.float32, device=dev)
        self._groups = RowGroups(max_tokens, top_k, self.experts, device=dev)

    def __call__(self, x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, out: Optional[torch.Tensor] = None,
                 stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """x bfloat16 [tokens][hidden], ids int32 and weights float32
        [tokens][top_k] from the router; returns [tokens][hidden] (bfloat16,
        or out's type).  The buffers serve one stream at a time."""
        what = "moe experts"
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
        check(lib.hi_rocm_moe_group(ids.data_ptr(), tokens, k, E, order, slots, offsets, st))
        check(lib.hi_rocm_moe_grouped_product(
            x.data_ptr(), tokens, x.stride(0) if tokens > 1 else H, order, k, offsets, places, E,
            self.w_up.data_ptr(), 2 * I, H, 1, h.data_ptr(), _CODES[h.dtype], I, st))
        check(lib.hi_rocm_moe_grouped_product(
            h.data_ptr(), places, I, 0, 1, offsets, places, E, self.w_down.data_ptr(), H, I, 0, y.data_ptr(),
            _CODES[y.dtype], H, st))
        check(lib.hi_rocm_moe_combine(
            y.data_ptr(), _CODES[y.dtype], H, slots, offsets, E, weights.data_ptr(), tokens, k, H, out.data_ptr(), code,
            out.stride(0) if tokens > 1 else H, st))
        return out


__all__ = ["RowGroups", "group_rows", "grouped_product", "combine", "MoeExperts"]

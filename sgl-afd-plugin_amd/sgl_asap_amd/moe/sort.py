"""A batch's tokens sorted by expert, and the experts' rows back to their tokens with the top-k weights applied.

The expert call does both inside (``afd_route``, ``afd_finalize``); here they stand alone, for experts that run elsewhere, and with
their gradients, for training. With pair p = t k + j, e the expert of ``topk_ids[t, j]`` less ``expert_lo`` (a pair whose e is
not in [0, num_experts), as of id -1, is not here)::

    positions[t, j] = how many pairs here come before p by (e, p), -1 if p is not here
    rows[positions[t, j]] = x[t]                               sort_tokens
    out[t] = sum_j topk_weights[t, j] rows[positions[t, j]]    unsort_tokens, in fp32, rounded once

Rows are [n k, hidden], in fp32, bf16 or fp16: the number that is used is known on the device alone (``offsets[-1]``).
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from .. import _lib
from .topk import fit_ints, last, launch, matrix_rows, need_gpu, no_tangent

VALUE_FORMATS = {torch.float32: _lib.AFD_V_F32, torch.bfloat16: _lib.AFD_V_BF16, torch.float16: _lib.AFD_V_F16}


def value_format(name: str, t: torch.Tensor) -> int:
    fmt = VALUE_FORMATS.get(t.dtype)
    if fmt is None:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return fmt


class TokenOrder(NamedTuple):
    """Where ``sort_tokens`` put the pairs."""

    positions: torch.Tensor  # i32 [n, k]: a pair's row, -1 if it is not here
    counts: torch.Tensor  # i32 [num_experts]: the experts' rows
    offsets: torch.Tensor  # i32 [num_experts + 1]: where they begin; the last: the rows that are used


class SortedOrder(TokenOrder):
    """The order that ``sort_tokens`` returns, every row before offsets[-1] being some pair's. Of what is made of it (a slice,
    ``_replace``, a copy), and of its tensors once they were changed, that is not known."""

    own = False  # whether sort_tokens made it

    @classmethod
    def made(cls, *tensors: torch.Tensor) -> "SortedOrder":
        order = cls(*tensors)
        order.own = True
        return order

    @classmethod
    def _make(cls, fields):
        return TokenOrder._make(fields)

    def __reduce__(self):
        return TokenOrder, tuple(self)

    def complete(self) -> bool:
        return self.own and not any(t.is_inference() or t._version for t in (self.positions, self.offsets))


@lru_cache(maxsize=1024)
def _workspace_bytes(n: int, k: int, experts: int) -> int:
    fit_ints(n, k, experts)
    out = ctypes.c_uint64()
    _lib.call("afd_sort_workspace", n, k, experts, ctypes.byref(out))
    return out.value


def _sort(x, ids, num_experts, expert_lo, out):
    """(rows, order) of ``afd_sort_tokens``."""
    (n, k), dev = ids.shape, x.device
    size = _workspace_bytes(n, k, num_experts)
    x, ldx = matrix_rows(x)
    hidden = x.shape[1]
    rows = torch.empty(n * k, hidden, dtype=x.dtype, device=dev) if out is None else out
    positions = torch.empty_like(ids)
    # tensors of their own: what adds up counts over ranks in place leaves the others as the backward saved them
    counts = torch.empty(num_experts, dtype=torch.int32, device=dev)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    # a call's own: calls on other streams and captured graphs each have theirs
    ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    ld = rows.stride(0) if rows.shape[0] > 1 else hidden
    launch("afd_sort_tokens", dev, VALUE_FORMATS[x.dtype], ids.data_ptr(), n, k, expert_lo, num_experts, x.data_ptr(), ldx, hidden,
           rows.data_ptr(), ld, out is None, positions.data_ptr(), counts.data_ptr(), offsets.data_ptr(),
           None if ws is None else ws.data_ptr(), size)
    return rows, SortedOrder.made(positions, counts, offsets)


def _unsort(rows, positions, weights):
    """``afd_unsort_tokens``."""
    (n, k), dev = positions.shape, rows.device
    rows, ld = matrix_rows(rows)
    out = torch.empty(n, rows.shape[1], dtype=rows.dtype, device=dev)
    launch("afd_unsort_tokens", dev, VALUE_FORMATS[rows.dtype], rows.data_ptr(), ld, rows.shape[0], positions.data_ptr(),
           None if weights is None else weights.data_ptr(), n, k, rows.shape[1], out.data_ptr())
    return out


class _Sort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, num_experts, expert_lo):
        rows, order = _sort(x, ids, num_experts, expert_lo, None)
        ctx.save_for_backward(order.positions)
        ctx.mark_non_differentiable(*order)
        ctx.set_materialize_grads(False)
        return (rows, *order)

    @staticmethod
    def backward(ctx, g, *_):
        if g is None:
            return None, None, None, None
        (positions,) = ctx.saved_tensors
        return last(_unsort(g, positions, None), g), None, None, None


class _Unsort(torch.autograd.Function):
    """rows as ``matrix_rows`` gives them: what the backward reads is then the input itself. offsets: None if there may be
    rows before the last that no pair has."""

    @staticmethod
    def forward(ctx, rows, weights, positions, offsets):
        need_w = weights is not None and ctx.needs_input_grad[1]
        ctx.save_for_backward(rows if need_w else None, weights, positions, offsets)
        ctx.rows = rows.shape
        ctx.set_materialize_grads(False)
        return _unsort(rows, positions, weights)

    @staticmethod
    def backward(ctx, g):
        if g is None:
            return None, None, None, None
        rows, weights, positions, offsets = ctx.saved_tensors
        (n, k), dev, (num_rows, hidden) = positions.shape, g.device, ctx.rows
        made_from = (g, rows, weights)
        g = g if g.is_contiguous() else g.contiguous()
        d_rows = d_w = None
        total = None
        if ctx.needs_input_grad[0]:
            # (without tokens no launch writes the rows; nor, of an order that is not complete, those that no pair has: those
            # past the last neither then, as positions may go there)
            d_rows = (torch.empty if n and offsets is not None else torch.zeros)(num_rows, hidden, dtype=g.dtype, device=dev)
            if offsets is None:
                offsets = torch.full((1,), 0x7FFFFFFF, dtype=torch.int32, device=dev)
            total = offsets.data_ptr() + 4 * (offsets.shape[0] - 1)
        if rows is not None:
            d_w = torch.empty(n, k, dtype=torch.float32, device=dev)
            rows, ld = matrix_rows(rows)
        else:
            ld = hidden
        launch("afd_unsort_grad", dev, VALUE_FORMATS[g.dtype], g.data_ptr(), None if rows is None else rows.data_ptr(), ld, num_rows,
               positions.data_ptr(), total, None if weights is None else weights.data_ptr(), n, k, hidden,
               None if d_rows is None else d_rows.data_ptr(), None if d_w is None else d_w.data_ptr())
        if torch.is_grad_enabled():
            d_rows, d_w = (None if t is None else last(t, *made_from) for t in (d_rows, d_w))
        return d_rows, d_w, None, None


def _matrix(name: str, t: torch.Tensor) -> None:
    if t.dim() != 2 or t.shape[1] < 1:
        raise ValueError(f"{name} must be [rows, hidden] with hidden >= 1, got {tuple(t.shape)}")
    if t.shape[1] > 0x7FFFFFFF:
        fit_ints(t.shape[1])
    value_format(name, t)


def sort_tokens(x: torch.Tensor, topk_ids: torch.Tensor, num_experts: int, *, expert_lo: int = 0,
                out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, TokenOrder]:
    """(rows [n k, hidden] sorted by expert, where they are) of tokens ``x`` [n, hidden] (fp32, bf16 or fp16) and ``topk_ids``
    int32 [n, k], for this rank's experts [expert_lo, expert_lo + num_experts), on the device's current stream.

    Rows past the last are 0. With ``out`` ([at least n k, hidden] in x's type, contiguous rows in memory that x's does not
    meet) the rows go there and those past the last stay as they are: what a serving rank that holds few of the experts
    uses, without a gradient; to autograd it is an in-place change of ``out``. An expert that a token names twice gets it twice.
    The rows have a gradient by x, once: second, forward-mode and traced derivatives are refused."""
    _matrix("x", x)
    if topk_ids.dtype != torch.int32 or topk_ids.dim() != 2:
        raise TypeError(f"topk_ids must be int32 [n, k], got {topk_ids.dtype} {tuple(topk_ids.shape)}")
    n, k = topk_ids.shape
    if x.shape[0] != n:
        raise ValueError(f"{n} rows of ids for x {tuple(x.shape)}")
    if n > 0x7FFFFFFF or k > 0x7FFFFFFF or not 0 <= num_experts <= 0x7FFFFFFF or not 0 <= expert_lo <= 0x7FFFFFFF:
        fit_ints(n, k, num_experts, expert_lo)
    need_gpu("x", x)
    if topk_ids.device != x.device:
        raise ValueError(f"topk_ids is on {topk_ids.device}, x on {x.device}")
    no_tangent("sort_tokens", x, out)
    ids = topk_ids if topk_ids.is_contiguous() else topk_ids.contiguous()
    if out is None:
        if torch.is_grad_enabled() and x.requires_grad:
            rows, *order = _Sort.apply(x, ids, num_experts, expert_lo)
            return rows, SortedOrder.made(*order)
        return _sort(x, ids, num_experts, expert_lo, None)
    if torch.is_grad_enabled() and (x.requires_grad or out.requires_grad):
        raise NotImplementedError("sort_tokens into out has no gradient: call it under torch.no_grad()")
    if out.dim() != 2 or out.dtype != x.dtype or out.shape[0] < n * k or out.shape[1] != x.shape[1]:
        raise ValueError(f"out must be {x.dtype} [at least {n * k}, {x.shape[1]}], got {out.dtype} {tuple(out.shape)}")
    if out.device != x.device or n > 0 and out.stride(1) != 1 or out.shape[0] > 1 and out.stride(0) < out.shape[1]:
        raise ValueError("out must have contiguous rows of its own on x's device")
    if _meet(x, out):
        raise ValueError("out meets x in memory")
    result = _sort(x, ids, num_experts, expert_lo, out)
    increment_version(out)  # a backward that saved what it held raises
    return result


def _meet(x: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether the memory from the first to the last element of both has a part in common (where x is read as it is)."""
    if x.numel() == 0 or out.numel() == 0 or matrix_rows(x)[0] is not x:
        return False
    ends = [t.data_ptr() + ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) * t.element_size() for t in (x, out)]
    return ends[0] > out.data_ptr() and ends[1] > x.data_ptr()


def unsort_tokens(rows: torch.Tensor, order: TokenOrder, topk_weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[n, hidden]: each token's sum of its ``rows`` [at least offsets[-1], hidden] (fp32, bf16 or fp16), with
    ``topk_weights`` [n, k] (fp32, others are cast; None: 1). Pairs that are not here add nothing, whatever their weights; a
    token without any gets 0. Added up in fp32 in the order of j, rounded once. Gradients by the rows (0 in those that no pair
    has) and the weights (0 where the pair is not here), once, as ``sort_tokens``.

    ``order`` may be one that was made of ``sort_tokens``': a part of the tokens' positions, or positions set to -1 to drop pairs
    (its gradient by the rows clears them first). A row is one pair's at most: two that name it would each write its gradient."""
    _matrix("rows", rows)
    positions, offsets = order.positions, order.offsets
    if positions.dtype != torch.int32 or positions.dim() != 2 or offsets.dtype != torch.int32 or offsets.dim() != 1:
        raise TypeError("order must hold int32 positions [n, k] and offsets [num_experts + 1]")
    n, k = positions.shape
    if n > 0x7FFFFFFF or k > 0x7FFFFFFF:
        fit_ints(n, k)
    need_gpu("rows", rows)
    dev = rows.device
    if positions.device != dev or offsets.device != dev or not positions.is_contiguous() or not offsets.is_contiguous():
        raise ValueError(f"positions and offsets must be contiguous on {dev}, got {positions.device} strides {positions.stride()} "
                         f"and {offsets.device} strides {offsets.stride()}")
    if offsets.shape[0] < 1:
        raise ValueError("offsets must hold the number of rows")
    no_tangent("unsort_tokens", rows, topk_weights)
    if topk_weights is not None:
        if topk_weights.shape != positions.shape or not topk_weights.is_floating_point():
            raise ValueError(f"topk_weights must be [{n}, {k}], got {topk_weights.dtype} {tuple(topk_weights.shape)}")
        if topk_weights.device != dev:
            raise ValueError(f"topk_weights is on {topk_weights.device}, rows on {dev}")
        if topk_weights.dtype != torch.float32 or not topk_weights.is_contiguous():
            topk_weights = topk_weights.to(torch.float32).contiguous()
    if torch.is_grad_enabled() and (rows.requires_grad or topk_weights is not None and topk_weights.requires_grad):
        whole = isinstance(order, SortedOrder) and order.complete()
        return _Unsort.apply(matrix_rows(rows)[0], topk_weights, positions, offsets if whole else None)
    return _unsort(rows, positions, topk_weights)

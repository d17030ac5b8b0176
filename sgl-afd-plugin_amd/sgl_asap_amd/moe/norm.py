"""The norms before and after a block, fused with its gate and the residual's scale (``afd_residual_norm``; the serving
engine's in the reference).

    rms(v) = v / sqrt(mean(v^2) + eps)                                  over the last dimension
    rms_norm:       rms(x) * weight                                     before a block
    residual_norm:  hidden = residual + scale * gate * (rms(y) * post_weight, or y)
                    normed = rms(hidden) * next_weight                  before the block behind it

y is the block's output. Activations are fp32, bf16 or fp16, the weights and the gate of the same type or fp32; everything
is computed in fp32 and rounded once (``normed`` is that of ``hidden`` before it is rounded). Values may be any numbers of
their type: a sum of squares past fp32 is made of scaled ones. The gradients, by every tensor, are one pass over the rows
too; sums over tokens run in a fixed order: the same call gives the same bits.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import NamedTuple, Optional

import torch

from .. import _lib
from .sort import value_format
from .topk import fit_ints, last, launch, matrix_rows, need_gpu, no_tangent

GATE_NONE, GATE_CHANNEL, GATE_TOKEN, GATE_ELEMENT = (_lib.AFD_GATE_NONE, _lib.AFD_GATE_CHANNEL, _lib.AFD_GATE_TOKEN,
                                                     _lib.AFD_GATE_ELEMENT)


class ResidualNorm(NamedTuple):
    hidden: torch.Tensor  # the residual stream behind the block
    normed: Optional[torch.Tensor]  # the next block's input, if next_weight was given


@lru_cache(maxsize=256)
def _cfg(columns: int, fmt: int, kind: int, post: bool, gate: bool, nxt: bool, scale: float, eps: float):
    return ctypes.pointer(_lib.AfdNormCfg(columns, fmt, kind, post, gate, nxt, scale, eps))


@lru_cache(maxsize=1024)
def _workspace_bytes(columns: int, n: int) -> int:
    out = ctypes.c_uint64()
    _lib.call("afd_residual_norm_workspace", _cfg(columns, 0, 0, False, False, False, 1.0, 1.0), n, ctypes.byref(out))
    return out.value


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _whole(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _forward(cfg, y, residual, w_post, gate, w_next, rstd):
    """(hidden or None, normed or None) of two-dimensional tensors."""
    residual, ldr = matrix_rows(residual)
    hidden = normed = y_ptr = h_ptr = n_ptr = next_ptr = None
    ldy = 0
    if y is not None:
        y, ldy = matrix_rows(y)
        hidden = _like(residual)
        y_ptr, h_ptr = y.data_ptr(), hidden.data_ptr()
    if w_next is not None:
        normed = _like(residual)
        n_ptr, next_ptr = normed.data_ptr(), w_next.data_ptr()
    launch("afd_residual_norm", residual.device, cfg, y_ptr, ldy, residual.data_ptr(), ldr, _ptr(w_post), _ptr(gate), next_ptr,
           residual.shape[0], h_ptr, n_ptr, _ptr(rstd))
    return hidden, normed


class _Norm(torch.autograd.Function):
    """y and residual two-dimensional, as ``matrix_rows`` gives them; without y the norm before a block alone."""

    @staticmethod
    def forward(ctx, y, residual, w_post, gate, w_next, cfg, kind):
        n = residual.shape[0]
        rstd = None
        if w_post is not None or w_next is not None:
            rstd = torch.empty(2, n, dtype=torch.float32, device=residual.device)
        hidden, normed = _forward(cfg, y, residual, w_post, gate, w_next, rstd)
        # the residual and y are read to make hidden again, y for its norm's gradient and the gate's too
        held = y if w_next is not None or w_post is not None or gate is not None and ctx.needs_input_grad[3] else None
        ctx.save_for_backward(held, residual if w_next is not None else None, w_post, gate, w_next, rstd)
        ctx.cfg, ctx.kind, ctx.shape, ctx.has_y, ctx.needs_next = cfg, kind, residual.shape, y is not None, w_next is not None
        ctx.set_materialize_grads(False)
        if y is None:
            return normed
        return (hidden, normed) if normed is not None else hidden

    @staticmethod
    def backward(ctx, *grads):
        dn = grads[-1] if ctx.needs_next else None
        dh = grads[0] if ctx.has_y else None
        if dh is None and dn is None:
            return (None,) * 7
        y, residual, w_post, gate, w_next, rstd = ctx.saved_tensors
        made_from = (dh, dn, y, residual, w_post, gate, w_next)
        need_y, need_res, need_post, need_gate, need_next, _, _ = ctx.needs_input_grad
        n, columns = ctx.shape
        dh_ptr = dn_ptr = y_ptr = res_ptr = d_y = d_res = d_post = d_gate = d_next = ws = None
        ldy = ldr = size = 0
        if dh is not None:
            g = dh = _whole(dh)
            dh_ptr = dh.data_ptr()
        if dn is not None:
            g = dn = _whole(dn)
            dn_ptr = dn.data_ptr()
            residual, ldr = matrix_rows(residual)
            res_ptr = residual.data_ptr()
        if y is not None:
            y, ldy = matrix_rows(y)
            y_ptr = y.data_ptr()
        dev = g.device
        # (without tokens no launch writes the parameters' gradients)
        like = torch.empty_like if n else torch.zeros_like
        if need_y:
            d_y = torch.empty_like(g)
        if need_res:
            d_res = torch.empty_like(g)
        if need_post:
            d_post = like(w_post)
        if need_gate:
            d_gate = like(gate)
        if need_next and dn is not None:
            d_next = like(w_next)
        if n:
            if d_post is not None or d_next is not None or d_gate is not None and ctx.kind == GATE_CHANNEL:
                size = _workspace_bytes(columns, n)
                ws = torch.empty(size, dtype=torch.uint8, device=dev)
            launch("afd_residual_norm_grad", dev, ctx.cfg, y_ptr, ldy, res_ptr, ldr, _ptr(w_post), _ptr(gate), _ptr(w_next),
                   _ptr(rstd), n, dh_ptr, dn_ptr, _ptr(d_res), _ptr(d_y), _ptr(d_gate), _ptr(d_post), _ptr(d_next), _ptr(ws), size)
        if torch.is_grad_enabled():
            d_y, d_res, d_post, d_gate, d_next = (None if t is None else last(t, *made_from)
                                                  for t in (d_y, d_res, d_post, d_gate, d_next))
        return d_y, d_res, d_post, d_gate, d_next, None, None


def _activations(name: str, t: torch.Tensor) -> int:
    fmt = value_format(name, t)
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} must be [..., hidden] with hidden >= 1, got {tuple(t.shape)}")
    fit_ints(t.shape[-1])
    return fmt


def _param(name: str, t: torch.Tensor, like: torch.Tensor, shape: tuple) -> bool:
    """Whether the parameter is held in fp32."""
    wide = t.dtype == torch.float32
    if not wide and t.dtype != like.dtype:
        raise TypeError(f"{name} must be {like.dtype} or float32, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, the activations on {like.device}")
    return wide


def _eps(eps: float) -> float:
    eps = float(eps)
    if not 0.0 < eps < float("inf"):
        raise ValueError(f"eps must be positive, got {eps}")
    return eps


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if t.dim() == 2 else t.reshape(-1, t.shape[-1])


def _needs_grad(*tensors: Optional[torch.Tensor]) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6) -> torch.Tensor:
    """``rms(x) * weight`` of ``x`` [..., hidden] (fp32, bf16 or fp16), in x's type, on the device's current stream. ``weight``
    [hidden] of x's type or fp32. Gradients by both, once: second, forward-mode and traced derivatives are refused."""
    fmt = _activations("x", x)
    columns = x.shape[-1]
    wide = _param("weight", weight, x, (columns,))
    need_gpu("x", x)
    no_tangent("rms_norm", x, weight)
    cfg = _cfg(columns, fmt, GATE_NONE, False, False, wide, 1.0, _eps(eps))
    weight, rows = _whole(weight), _rows(x)
    if _needs_grad(x, weight):
        out = _Norm.apply(None, matrix_rows(rows)[0], None, None, weight, cfg, GATE_NONE)
    else:
        out = _forward(cfg, None, rows, None, None, weight, None)[1]
    return out if rows is x else out.view(x.shape)


def residual_norm(
    y: torch.Tensor,
    residual: torch.Tensor,
    *,
    post_weight: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    scale: float = 1.0,
    next_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
) -> ResidualNorm:
    """(hidden, normed) of a block's output ``y`` and the ``residual`` it is added to, both [..., hidden] in one type (fp32,
    bf16 or fp16), on the device's current stream.

    ``post_weight`` [hidden]: the norm after the block (None: none). ``gate``: [hidden], one value per channel, [..., 1], per
    token, or [..., hidden], per element. ``scale``: a number. ``next_weight`` [hidden]: the norm before the block behind it
    (None: ``normed`` is None). Weights and gate are of y's type or fp32. Gradients by every tensor, once: second, forward-mode and
    traced derivatives are refused."""
    fmt = _activations("y", y)
    if residual.dtype != y.dtype or residual.shape != y.shape:
        raise ValueError(f"y is {y.dtype} {tuple(y.shape)}, residual {residual.dtype} {tuple(residual.shape)}")
    if residual.device != y.device:
        raise ValueError(f"residual is on {residual.device}, y on {y.device}")
    columns, kind = y.shape[-1], GATE_NONE
    wide_post = wide_gate = wide_next = False
    if post_weight is not None:
        wide_post = _param("post_weight", post_weight, y, (columns,))
        post_weight = _whole(post_weight)
    if next_weight is not None:
        wide_next = _param("next_weight", next_weight, y, (columns,))
        next_weight = _whole(next_weight)
    if gate is not None:
        if gate.dim() == 1 and (y.dim() > 1 or gate.shape[0] == columns):  # ([1] beside one token: its gate)
            kind, wide_gate = GATE_CHANNEL, _param("gate", gate, y, (columns,))
        elif gate.shape == y.shape and columns > 1:
            kind, wide_gate = GATE_ELEMENT, _param("gate", gate, y, tuple(y.shape))
            gate = _rows(gate)
        else:
            kind, wide_gate = GATE_TOKEN, _param("gate", gate, y, tuple(y.shape[:-1]) + (1,))
            gate = gate.reshape(-1)
        gate = _whole(gate)
    need_gpu("y", y)
    no_tangent("residual_norm", y, residual, post_weight, gate, next_weight)
    cfg = _cfg(columns, fmt, kind, wide_post, wide_gate, wide_next, float(scale), _eps(eps))
    rows = _rows(y)
    if _needs_grad(y, residual, post_weight, gate, next_weight):
        out = _Norm.apply(matrix_rows(rows)[0], matrix_rows(_rows(residual))[0], post_weight, gate, next_weight, cfg, kind)
        hidden, normed = out if next_weight is not None else (out, None)
    else:
        hidden, normed = _forward(cfg, rows, _rows(residual), post_weight, gate, next_weight, None)
    if rows is not y:
        hidden, normed = hidden.view(y.shape), None if normed is None else normed.view(y.shape)
    return ResidualNorm(hidden, normed)


class BlockNorms(torch.nn.Module):
    """A block's norms, gate and residual scale as a module: ``hidden = residual + scale * gate * rms(y) * post_weight``.

    ``input_weight`` [hidden]: the norm before the block (``before``); ``post_weight``: after it (None: none); ``gate``
    [hidden]: learned per channel (None: none). They are parameters: those that are given as one are the module's own."""

    def __init__(self, input_weight: torch.Tensor, post_weight: Optional[torch.Tensor] = None,
                 gate: Optional[torch.Tensor] = None, scale: float = 1.0, eps: float = 1e-6):
        super().__init__()
        for name, t in (("input_weight", input_weight), ("post_weight", post_weight), ("gate", gate)):
            if t is not None and (t.dim() != 1 or t.shape != input_weight.shape):
                raise ValueError(f"{name} must be {tuple(input_weight.shape)}, got {tuple(t.shape)}")
            self.register_parameter(name, t if t is None or isinstance(t, torch.nn.Parameter) else torch.nn.Parameter(t))
        self.scale, self.eps = float(scale), _eps(eps)

    def before(self, x: torch.Tensor) -> torch.Tensor:
        return rms_norm(x, self.input_weight, eps=self.eps)

    def after(self, y: torch.Tensor, residual: torch.Tensor, gate: Optional[torch.Tensor] = None,
              next_weight: Optional[torch.Tensor] = None) -> ResidualNorm:
        """``gate``: in place of the learned one (per token or per element, from the tokens)."""
        return residual_norm(y, residual, post_weight=self.post_weight, gate=self.gate if gate is None else gate,
                             scale=self.scale, next_weight=next_weight, eps=self.eps)

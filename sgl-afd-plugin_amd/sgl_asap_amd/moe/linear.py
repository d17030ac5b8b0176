"""A dense layer with block-FP8 weights: ``y = bf16(q(x) W^T)``, W in e4m3 with one fp32 scale per 128x128 block, x
quantized in the call to e4m3 with one fp32 scale per 1x128 (``afd_linear``).

The format is the experts' (FP8 checkpoints hold their dense layers in it too, the
shared expert's among them); the reference leaves these layers to the serving engine. Any sizes, one token to prefill.
For serving: the product has no gradient.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache
from typing import Optional

import torch

from .. import _lib
from .topk import fit_ints, launch, matrix_rows, need_gpu, no_tangent

FP8_BLOCK = 128


@lru_cache(maxsize=1024)
def _workspace_bytes(n: int, k_in: int) -> int:
    out = ctypes.c_uint64()
    _lib.call("afd_linear_workspace", n, k_in, ctypes.byref(out))
    return out.value


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether rows of a and b (of one length in bytes an element) may share an element."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    n, size = a.shape[0], a.element_size()
    ends = [t.data_ptr() + ((n - 1) * t.stride(0) + t.shape[1]) * size for t in (a, b)]
    if ends[0] <= b.data_ptr() or ends[1] <= a.data_ptr():
        return False
    # columns of one buffer: b's begin behind a's and end before the next row's
    if n > 1 and a.stride(0) == b.stride(0):
        at = (b.data_ptr() - a.data_ptr()) % (a.stride(0) * size)
        return at < a.shape[1] * size or at + b.shape[1] * size > a.stride(0) * size
    return True


class Fp8BlockLinear(torch.nn.Module):
    """``weight``: e4m3 codes [n_out, k_in] (float8_e4m3fn, or their bytes); ``scales``: fp32
    [ceil(n_out / 128), ceil(k_in / 128)], the weight being code x scale. Laid out once for the kernels, on ``device``
    (default: the codes'), where the layer stays: moves and casts of a module leave it, and like the bf16 MLP's weights its own
    are not in ``state_dict()`` (they come from the checkpoint). It can be copied and pickled."""

    def __init__(self, weight: torch.Tensor, scales: torch.Tensor, device=None):
        super().__init__()
        if weight.dim() != 2 or weight.dtype not in (torch.float8_e4m3fn, torch.uint8, torch.int8):
            raise TypeError(f"expected e4m3 codes [n_out, k_in], got {weight.dtype} {tuple(weight.shape)}")
        n_out, k_in = weight.shape
        blocks = (-(-n_out // FP8_BLOCK), -(-k_in // FP8_BLOCK))
        if scales.dtype != torch.float32 or tuple(scales.shape) != blocks:
            raise ValueError(f"scales must be float32 {blocks} for weights {n_out} x {k_in}, got {scales.dtype} "
                             f"{tuple(scales.shape)}")
        fit_ints(n_out, k_in)
        size = ctypes.c_uint64()
        _lib.call("afd_linear_layout", n_out, k_in, ctypes.byref(size))
        device = torch.device(device) if device is not None else weight.device
        codes = weight.contiguous().view(torch.uint8).to(device)
        need_gpu("weight", codes)
        self.out_features, self.in_features = n_out, k_in
        self.image = torch.empty(size.value, dtype=torch.uint8, device=codes.device)
        self.scales = scales.to(codes.device, copy=True).contiguous()
        launch("afd_linear_pack", codes.device, codes.data_ptr(), k_in, n_out, k_in, self.image.data_ptr())
        self._point()

    def _point(self) -> None:
        # _weights holds addresses: the tensors stay attributes, not buffers that a module move would replace
        self._weights = _lib.AfdLinearWeights(self.out_features, self.in_features, self.image.data_ptr(), self.scales.data_ptr())
        self._weights_ref = ctypes.byref(self._weights)

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("_weights", "_weights_ref")}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._point()

    def forward(self, x: torch.Tensor, out: Optional[torch.Tensor] = None, *, silu_mul: bool = False) -> torch.Tensor:
        """bf16 [..., k_in] -> bf16 [..., n_out] on the device's current stream, into ``out`` if given ([n,
        n_out] with contiguous rows that share no element with x, x two-dimensional). ``silu_mul``: as the method."""
        if silu_mul:
            return self._product("afd_linear_silu_mul", x, 2 * self.in_features, out)
        return self._product("afd_linear", x, self.in_features, out)

    def silu_mul(self, gate_up: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The layer of ``silu_mul(gate_up)``, bf16 [..., 2 k_in] of [gate | up] rows, bit for bit, in a launch less and
        without the activation in memory. A call of the module: its hooks run, and see gate_up as what goes in."""
        return self(gate_up, out, silu_mul=True)

    def _product(self, name, x, columns, out):
        if x.dtype != torch.bfloat16 or x.dim() < 1 or x.shape[-1] != columns:
            raise TypeError(f"expected bf16 [..., {columns}], got {x.dtype} {tuple(x.shape)}")
        if x.device != self.image.device:
            raise ValueError(f"x is on {x.device}, the weights on {self.image.device}")
        if torch.is_grad_enabled() and (x.requires_grad or out is not None and out.requires_grad):
            raise NotImplementedError("Fp8BlockLinear has no gradient: call it under torch.no_grad()")
        no_tangent("Fp8BlockLinear", x, out)
        rows = x if x.dim() == 2 else x.reshape(-1, columns)
        rows, ldx = matrix_rows(rows)
        n = rows.shape[0]
        if out is None:
            y = torch.empty(n, self.out_features, dtype=torch.bfloat16, device=x.device)
        else:
            y = out
            if x.dim() != 2 or y.dtype != torch.bfloat16 or tuple(y.shape) != (n, self.out_features):
                raise ValueError(f"out must be bf16 [{n}, {self.out_features}] for a two-dimensional x, got {y.dtype} "
                                 f"{tuple(y.shape)}")
            if y.device != x.device or n > 0 and y.stride(1) != 1 or n > 1 and y.stride(0) < self.out_features:
                raise ValueError("out must have contiguous rows of its own on x's device")
            if _overlap(rows, y):
                raise ValueError("out shares elements with x")
        size = _workspace_bytes(n, self.in_features)
        # a call's own: calls on other streams and captured graphs each have theirs
        ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        launch(name, x.device, self._weights_ref, rows.data_ptr(), ldx, n,
               ws.data_ptr(), size, y.data_ptr(), y.stride(0) if n > 1 else self.out_features)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], self.out_features)

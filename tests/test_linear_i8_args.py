"""Refusals of the dense int8 product, on the host."""

import ctypes

import pytest
import torch

from sgl_asap_amd import _lib
from sgl_asap_amd.moe.linear import Int8Linear
from sgl_asap_amd.moe.shared import Int8SharedExpertMLP

OK, ARG, SHAPE, WS = _lib.AFD_OK, _lib.AFD_ERR_ARG, _lib.AFD_ERR_SHAPE, _lib.AFD_ERR_WORKSPACE


def test_sizes():
    L, out = _lib.lib(), ctypes.c_uint64()
    assert L.afd_linear_i8_workspace(1, 1, None) == ARG
    assert L.afd_linear_i8_workspace(-1, 1, ctypes.byref(out)) == ARG
    assert L.afd_linear_i8_workspace((1 << 22) + 1, 1, ctypes.byref(out)) == ARG
    for k in (0, -1, 65537):
        assert L.afd_linear_i8_workspace(1, k, ctypes.byref(out)) == SHAPE
    assert L.afd_linear_i8_workspace(17, 130, ctypes.byref(out)) == OK
    assert out.value >= 32 * 256 + 32 * 4


@pytest.mark.parametrize("silu", [False, True])
def test_calls(silu):
    L = _lib.lib()
    entry = L.afd_linear_i8_silu_mul if silu else L.afd_linear_i8
    wide = 400 if silu else 200

    def call(n=4, ldx=wide, ldy=100, x=16, ws=16, size=1 << 30, y=16, n_out=100, k=200, image=16, scales=16):
        w = _lib.AfdLinearWeights(n_out, k, image, scales)
        return entry(ctypes.byref(w), x, ldx, n, ws, size, y, ldy, None)

    assert call(n=0) == OK and call(n=0, x=None, y=None, ws=None) == OK
    assert entry(None, 16, wide, 4, 16, 1 << 30, 16, 100, None) == ARG
    assert call(n=-1) == ARG and call(n=(1 << 22) + 1) == ARG
    for name in ("x", "ws", "y", "image", "scales"):
        assert call(**{name: None}) == ARG, name
    assert call(ldx=wide - 1) == SHAPE and call(ldy=99) == SHAPE and call(n_out=0) == SHAPE
    assert call(k=70000, ldx=140000) == SHAPE and call(n_out=70000, ldy=70000) == SHAPE
    assert call(image=24) == SHAPE and call(ws=24) == WS
    need = ctypes.c_uint64()
    assert L.afd_linear_i8_workspace(4, 200, ctypes.byref(need)) == OK
    assert call(size=need.value - 1) == WS


def test_python_refusals():
    codes, scales = torch.zeros(130, 200, dtype=torch.int8), torch.zeros(130)
    with pytest.raises(ValueError, match="GPU"):
        Int8Linear(codes, scales)
    for bad in (codes.float(), codes[0], codes.to(torch.uint8), codes[None]):
        with pytest.raises(TypeError):
            Int8Linear(bad, scales)
    for bad in (scales[:129], scales.double(), scales[None], torch.zeros(130, 2), torch.zeros(())):
        with pytest.raises(ValueError):
            Int8Linear(codes, bad)
    for shape in ((130, 64), (64, 12)):
        with pytest.raises(ValueError):
            Int8SharedExpertMLP(torch.zeros(shape[0] if shape[1] == 64 else 24, 64, dtype=torch.int8), scales,
                                torch.zeros(64, 64 if shape[1] == 64 else 13, dtype=torch.int8), scales)


def test_sizes_past_32_bits_are_refused(monkeypatch):
    from sgl_asap_amd.moe import linear as M

    called, big = [], (1 << 32) + 8
    monkeypatch.setattr(M, "need_gpu", lambda *a: None)
    monkeypatch.setattr(M, "launch", lambda *a: called.append(a))
    for n_out, k in ((big, 1), (1, big)):
        with pytest.raises(ValueError, match="32 bits"):
            Int8Linear(torch.empty(n_out, k, dtype=torch.int8, device="meta"), torch.empty(n_out, device="meta"))
    layer = Int8Linear(torch.zeros(4, 2, dtype=torch.int8), torch.zeros(4))
    layer.image = layer.image.to("meta")
    called.clear()
    with pytest.raises(ValueError, match="32 bits"):
        layer(torch.empty(big, 2, dtype=torch.bfloat16, device="meta"))
    with pytest.raises(ValueError, match="32 bits"):
        layer.silu_mul(torch.empty(big, 4, dtype=torch.bfloat16, device="meta"))
    assert not called

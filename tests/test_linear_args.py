"""Refusals of the dense FP8 block product, on the host."""

import ctypes

import pytest
import torch

from sgl_asap_amd import _lib
from sgl_asap_amd.moe.linear import Fp8BlockLinear
from sgl_asap_amd.moe.shared import Fp8SharedExpertMLP

OK, ARG, SHAPE, WS = _lib.AFD_OK, _lib.AFD_ERR_ARG, _lib.AFD_ERR_SHAPE, _lib.AFD_ERR_WORKSPACE


def test_sizes():
    L, out = _lib.lib(), ctypes.c_uint64()
    assert L.afd_linear_layout(1, 1, ctypes.byref(out)) == OK and out.value == 16 * 128
    assert L.afd_linear_layout(4097, 2000, ctypes.byref(out)) == OK and out.value == 4112 * 2048
    for n_out, k in ((0, 1), (1, 0), (65537, 1), (1, 65537), (-1, 4)):
        assert L.afd_linear_layout(n_out, k, ctypes.byref(out)) == SHAPE
        assert L.afd_linear_pack(16, 65537, n_out, k, 16, None) == SHAPE
    assert L.afd_linear_layout(1, 1, None) == ARG and L.afd_linear_workspace(1, 1, None) == ARG
    assert L.afd_linear_workspace(-1, 1, ctypes.byref(out)) == ARG
    assert L.afd_linear_workspace((1 << 22) + 1, 1, ctypes.byref(out)) == ARG
    assert L.afd_linear_workspace(1, 0, ctypes.byref(out)) == SHAPE
    assert L.afd_linear_workspace(17, 130, ctypes.byref(out)) == OK
    assert out.value == 32 * 256 + 2 * 256 * 4
    assert L.afd_linear_pack(None, 16, 4, 16, 16, None) == ARG and L.afd_linear_pack(16, 16, 4, 16, None, None) == ARG
    assert L.afd_linear_pack(16, 15, 4, 16, 16, None) == SHAPE and L.afd_linear_pack(16, 16, 4, 16, 24, None) == SHAPE


def test_calls():
    L = _lib.lib()

    def call(n=4, ldx=200, ldy=100, x=16, ws=16, size=1 << 30, y=16, n_out=100, k=200, image=16, scales=16):
        w = _lib.AfdLinearWeights(n_out, k, image, scales)
        return L.afd_linear(ctypes.byref(w), x, ldx, n, ws, size, y, ldy, None)

    assert call(n=0) == OK and call(n=0, x=None, y=None, ws=None) == OK
    assert L.afd_linear(None, 16, 200, 4, 16, 1 << 30, 16, 100, None) == ARG
    assert call(n=-1) == ARG and call(n=(1 << 22) + 1) == ARG
    for name in ("x", "ws", "y", "image", "scales"):
        assert call(**{name: None}) == ARG, name
    assert call(ldx=199) == SHAPE and call(ldy=99) == SHAPE and call(n_out=0) == SHAPE and call(k=70000, ldx=70000) == SHAPE
    assert call(image=24) == SHAPE and call(ws=24) == WS
    need = ctypes.c_uint64()
    assert L.afd_linear_workspace(4, 200, ctypes.byref(need)) == OK
    assert call(size=need.value - 1) == WS


def test_python_refusals():
    codes, scales = torch.zeros(130, 200, dtype=torch.uint8), torch.zeros(2, 2)
    with pytest.raises(ValueError, match="GPU"):
        Fp8BlockLinear(codes, scales)
    with pytest.raises(TypeError):
        Fp8BlockLinear(codes.float(), scales)
    with pytest.raises(TypeError):
        Fp8BlockLinear(codes[0], scales)
    with pytest.raises(ValueError):
        Fp8BlockLinear(codes, torch.zeros(1, 2))
    with pytest.raises(ValueError):
        Fp8BlockLinear(codes, scales.double())
    with pytest.raises(ValueError):
        Fp8SharedExpertMLP(torch.zeros(130, 64, dtype=torch.uint8), scales, torch.zeros(64, 64, dtype=torch.uint8), scales)
    with pytest.raises(ValueError):
        Fp8SharedExpertMLP(torch.zeros(24, 64, dtype=torch.uint8), scales, torch.zeros(64, 12, dtype=torch.uint8), scales)


@pytest.mark.gpu
def test_python_refusals_of_calls():
    layer = Fp8BlockLinear(torch.zeros(130, 200, dtype=torch.uint8, device="cuda"), torch.zeros(2, 2, device="cuda"))
    x = torch.zeros(4, 200, dtype=torch.bfloat16, device="cuda")
    for bad in (x.float(), x[:, :199], torch.zeros((), dtype=torch.bfloat16, device="cuda")):
        with pytest.raises(TypeError):
            layer(bad)
    with pytest.raises(ValueError):
        layer(x.cpu())
    with pytest.raises(NotImplementedError):
        layer(x.clone().requires_grad_())
    for out in (torch.empty(4, 129, dtype=torch.bfloat16, device="cuda"), torch.empty(4, 130, device="cuda"),
                torch.empty(130, 4, dtype=torch.bfloat16, device="cuda").t(),
                torch.empty(1, 130, dtype=torch.bfloat16, device="cuda").expand(4, 130)):
        with pytest.raises(ValueError):
            layer(x, out=out)
    with pytest.raises(ValueError):
        layer(x.view(2, 2, 200), out=torch.empty(4, 130, dtype=torch.bfloat16, device="cuda"))


def test_overlap():
    from sgl_asap_amd.moe.linear import _overlap

    buf = torch.zeros(10, 48, dtype=torch.bfloat16)
    x = buf[2:6, 8:24]
    apart = [buf[2:6, 24:48], buf[2:6, :8], buf[1:5, 24:40], buf[3:7, 24:30], buf[6:10, 8:24], torch.zeros(4, 16), buf[2:2, :]]
    shared = [x, buf[2:6, 23:30], buf[2:6, :9], buf[1:5, 8:24], buf[3:7, 0:48], buf[5:9, 8:24], buf.view(5, 96)[1:3, :16]]
    for y in apart:
        assert not _overlap(x[: y.shape[0]], y) and not _overlap(y, x[: y.shape[0]])
    for y in shared:
        assert _overlap(x[: y.shape[0]], y) and _overlap(y, x[: y.shape[0]])
    one = buf[3:4, :16]
    assert not _overlap(one, buf[3:4, 16:40]) and _overlap(one, buf[3:4, 15:40])


def test_silu_mul_calls():
    L = _lib.lib()

    def call(n=4, ld=400, x=16, ws=16, size=1 << 30, y=16, ldy=100, image=16):
        w = _lib.AfdLinearWeights(100, 200, image, 16)
        return L.afd_linear_silu_mul(ctypes.byref(w), x, ld, n, ws, size, y, ldy, None)

    assert call(n=0) == OK and call(n=0, x=None, y=None, ws=None) == OK
    assert L.afd_linear_silu_mul(None, 16, 400, 4, 16, 1 << 30, 16, 100, None) == ARG
    assert call(n=-1) == ARG and call(x=None) == ARG and call(y=None) == ARG and call(ws=None) == ARG and call(image=None) == ARG
    assert call(ld=399) == SHAPE and call(ldy=99) == SHAPE and call(image=24) == SHAPE
    assert call(ws=24) == WS and call(size=100) == WS


def test_sizes_past_32_bits_are_refused(monkeypatch):
    """Sizes are C ints at the entry points: one past their range must not come out as another, smaller one."""
    from sgl_asap_amd.moe import linear as M

    called, big = [], (1 << 32) + 8
    monkeypatch.setattr(M, "need_gpu", lambda *a: None)
    monkeypatch.setattr(M, "launch", lambda *a: called.append(a))
    for n_out, k in ((big, 1), (1, big)):
        with pytest.raises(ValueError, match="32 bits"):
            Fp8BlockLinear(torch.empty(n_out, k, dtype=torch.uint8, device="meta"),
                           torch.empty(-(-n_out // 128), -(-k // 128), device="meta"))
    layer = Fp8BlockLinear(torch.zeros(4, 2, dtype=torch.uint8), torch.zeros(1, 1))
    layer.image = layer.image.to("meta")
    called.clear()
    for x in (torch.empty(big, 2, dtype=torch.bfloat16, device="meta"), torch.empty(2, big // 2, 2, dtype=torch.bfloat16, device="meta")):
        with pytest.raises(ValueError, match="32 bits"):
            layer(x)
    with pytest.raises(ValueError, match="32 bits"):
        layer.silu_mul(torch.empty(big, 4, dtype=torch.bfloat16, device="meta"))
    assert not called

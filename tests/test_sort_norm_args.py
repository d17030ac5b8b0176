"""Refusals of the sorted tokens and of a block's norms, on the host."""

import ctypes

import pytest
import torch

from sgl_asap_amd import _lib
from sgl_asap_amd.moe.layer import AsapMoE
from sgl_asap_amd.moe.norm import BlockNorms, residual_norm, rms_norm
from sgl_asap_amd.moe.sort import TokenOrder, sort_tokens, unsort_tokens

OK, ARG, SHAPE, FMT, WS = (_lib.AFD_OK, _lib.AFD_ERR_ARG, _lib.AFD_ERR_SHAPE, _lib.AFD_ERR_UNSUPPORTED,
                           _lib.AFD_ERR_WORKSPACE)


def test_sort_workspace():
    L, out = _lib.lib(), ctypes.c_uint64(77)
    size = lambda *a: L.afd_sort_workspace(*a, ctypes.byref(out))  # noqa: E731
    assert size(0, 1, 1) == OK and out.value == 0
    assert size(512, 8, 1024) == OK and out.value == 0
    assert size(513, 8, 64) == OK and out.value == 5 * 64 * 4
    assert size(1 << 26, 31, 1024) == OK and out.value <= 256 * 1024 * 4
    assert L.afd_sort_workspace(1, 1, 1, None) == ARG
    assert size(-1, 1, 1) == ARG and size((1 << 26) + 1, 1, 1) == ARG
    for bad in ((1, 0, 1), (1, 33, 1), (1, 1, 0), (1, 1, 1025), (1 << 26, 32, 4)):
        assert size(*bad) == SHAPE, bad


def test_sort_calls():
    L = _lib.lib()

    def sort(fmt=1, ids=16, n=600, k=8, lo=0, experts=4, x=16, ldx=10, columns=10, rows=16, ld=10, zero=1, pos=16, counts=16,
             offsets=16, ws=16, size=1 << 20):
        return L.afd_sort_tokens(fmt, ids, n, k, lo, experts, x, ldx, columns, rows, ld, zero, pos, counts, offsets, ws, size, None)

    for name in ("ids", "x", "rows", "pos", "counts", "offsets"):
        assert sort(**{name: None}) == ARG, name
    assert sort(fmt=3) == FMT and sort(fmt=-1) == FMT
    assert sort(lo=-1) == ARG and sort(n=-1) == ARG and sort(k=0) == SHAPE and sort(k=33) == SHAPE and sort(experts=0) == SHAPE
    assert sort(experts=1025) == SHAPE and sort(columns=0) == SHAPE and sort(columns=65537, ldx=65537, ld=65537) == SHAPE
    assert sort(ldx=9) == SHAPE and sort(ld=9) == SHAPE
    assert sort(ws=None) == WS and sort(size=5 * 4 * 4 - 1) == WS and sort(ws=18) == WS

    def back(fmt=1, rows=16, ld=10, num=20, pos=16, w=None, n=5, k=4, columns=10, out=16):
        return L.afd_unsort_tokens(fmt, rows, ld, num, pos, w, n, k, columns, out, None)

    assert back(n=0) == OK and back(n=0, rows=None, pos=None, out=None) == OK
    for name in ("rows", "pos", "out"):
        assert back(**{name: None}) == ARG, name
    assert back(fmt=4) == FMT and back(ld=9) == SHAPE and back(num=-1) == SHAPE and back(k=40) == SHAPE and back(n=-2) == ARG

    def grad(fmt=1, g=16, rows=16, ld=10, num=20, pos=16, total=16, w=None, n=5, k=4, columns=10, d_rows=16, d_w=16):
        return L.afd_unsort_grad(fmt, g, rows, ld, num, pos, total, w, n, k, columns, d_rows, d_w, None)

    assert grad(n=0) == OK and grad(d_rows=None, d_w=None) == OK
    for name in ("g", "rows", "pos", "total"):
        assert grad(**{name: None}) == ARG, name
    assert grad(fmt=7) == FMT and grad(ld=9) == SHAPE and grad(num=-1) == SHAPE and grad(n=-1) == ARG


def test_norm_calls():
    L, out = _lib.lib(), ctypes.c_uint64()

    def cfg(columns=64, fmt=1, kind=0, scale=1.0, eps=1e-6):
        return ctypes.byref(_lib.AfdNormCfg(columns, fmt, kind, 0, 0, 0, scale, eps))

    def call(c=None, y=16, ldy=64, res=16, ldr=64, post=None, gate=None, nxt=None, n=4, h=16, normed=None, rstd=None):
        return L.afd_residual_norm(c or cfg(), y, ldy, res, ldr, post, gate, nxt, n, h, normed, rstd, None)

    def bad_cfgs(f):
        assert f(cfg(columns=0)) == SHAPE and f(cfg(columns=16385)) == SHAPE
        assert f(cfg(fmt=3)) == FMT and f(cfg(kind=4)) == FMT and f(cfg(kind=-1)) == FMT
        assert f(cfg(eps=0.0)) == ARG and f(cfg(eps=float("nan"))) == ARG and f(cfg(eps=-1.0)) == ARG

    bad_cfgs(lambda c: call(c, ldy=1 << 20, ldr=1 << 20))
    assert L.afd_residual_norm(None, 16, 64, 16, 64, None, None, None, 4, 16, None, None, None) == ARG
    assert call(n=0) == OK and call(n=0, y=None, res=None, h=None) == OK
    assert call(n=-1) == ARG and call(res=None) == ARG and call(h=None) == ARG and call(y=None) == ARG
    assert call(normed=16) == ARG and call(cfg(kind=2)) == ARG
    assert call(ldy=63) == SHAPE and call(ldr=63) == SHAPE

    bad_cfgs(lambda c: L.afd_residual_norm_workspace(c, 4, ctypes.byref(out)))
    assert L.afd_residual_norm_workspace(cfg(), 4, None) == ARG
    assert L.afd_residual_norm_workspace(cfg(), 0, ctypes.byref(out)) == OK and out.value == 0
    assert L.afd_residual_norm_workspace(cfg(), 1 << 26, ctypes.byref(out)) == OK and 0 < out.value < 1 << 26

    def grad(c=None, y=16, ldy=64, h=16, ldh=64, post=None, gate=None, nxt=16, rstd=16, n=4, dh=16, dn=16, d_res=16, d_y=16,
             d_gate=None, d_post=None, d_next=16, ws=16, size=1 << 30):
        return L.afd_residual_norm_grad(c or cfg(), y, ldy, h, ldh, post, gate, nxt, rstd, n, dh, dn, d_res, d_y, d_gate, d_post,
                                        d_next, ws, size, None)

    bad_cfgs(lambda c: grad(c, ldy=1 << 20, ldh=1 << 20))
    assert grad(n=0) == OK
    assert grad(dh=None, dn=None, d_next=None) == ARG and grad(h=None) == ARG and grad(nxt=None) == ARG and grad(rstd=None) == ARG
    assert grad(dn=None) == ARG  # d_next without dn
    assert grad(d_post=16) == ARG and grad(d_gate=16) == ARG and grad(cfg(kind=1)) == ARG
    assert grad(y=None, post=16) == ARG and grad(y=None) == ARG and grad(cfg(kind=1), y=None, gate=16, d_gate=16) == ARG
    assert grad(ldy=63) == SHAPE and grad(ldh=63) == SHAPE
    assert grad(ws=None) == WS and grad(size=16) == WS and grad(ws=24) == WS


def test_python_refusals_of_sort():
    x, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        sort_tokens(x, ids, 4)
    for bad in (x.double(), x.to(torch.int32)):
        with pytest.raises(TypeError):
            sort_tokens(bad, ids, 4)
    for bad in (x[0], x[None], x[:, :0]):
        with pytest.raises(ValueError):
            sort_tokens(bad, ids, 4)
    for bad in (ids.long(), ids[0], ids.float()):
        with pytest.raises(TypeError):
            sort_tokens(x, bad, 4)
    with pytest.raises(ValueError):
        sort_tokens(x[:3], ids, 4)
    for experts, lo in ((1 << 32, 0), (4, 1 << 31)):
        with pytest.raises(ValueError, match="32 bits"):
            sort_tokens(x, ids, experts, expert_lo=lo)
    order = TokenOrder(ids, ids[0], torch.zeros(5, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        unsort_tokens(x, order)
    for bad in (TokenOrder(ids.long(), ids[0], order.offsets), TokenOrder(ids[0], ids[0], order.offsets),
                TokenOrder(ids, ids[0], order.offsets.long()), TokenOrder(ids, ids[0], order.offsets[None])):
        with pytest.raises(TypeError):
            unsort_tokens(x, bad)


def test_python_refusals_of_norms():
    x, w = torch.zeros(4, 8), torch.zeros(8)
    for call in (lambda: rms_norm(x, w), lambda: residual_norm(x, x)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for call in (lambda: rms_norm(x.double(), w), lambda: rms_norm(x, w.to(torch.bfloat16)), lambda: rms_norm(x, w.double()),
                 lambda: residual_norm(x.int(), x.int()), lambda: residual_norm(x, x, gate=w.half())):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: rms_norm(x, w[:7]), lambda: rms_norm(x, w[None]), lambda: rms_norm(torch.zeros(()), w),
                 lambda: rms_norm(x[:, :0], w[:0]), lambda: rms_norm(x, w, eps=0.0), lambda: rms_norm(x, w, eps=float("nan")),
                 lambda: residual_norm(x, x[:3]), lambda: residual_norm(x, x.half()), lambda: residual_norm(x, x, gate=w[:1]),
                 lambda: residual_norm(x, x, gate=x[:3]), lambda: residual_norm(x, x, gate=x[:, :2]),
                 lambda: residual_norm(x, x, gate=torch.zeros(())), lambda: residual_norm(x, x, post_weight=w[:4]),
                 lambda: residual_norm(x, x, next_weight=w[:4]), lambda: BlockNorms(w, w[:4]), lambda: BlockNorms(x),
                 lambda: BlockNorms(w, eps=0.0)):
        with pytest.raises(ValueError):
            call()


def test_layer_refuses_a_residual_without_norms():
    layer = AsapMoE(8, 16, 16, 0)
    for kw in (dict(residual=torch.zeros(1, 16)), dict(next_weight=torch.zeros(16))):
        with pytest.raises(ValueError, match="norms"):
            layer(torch.zeros(1, 16), None, **kw)

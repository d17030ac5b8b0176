"""Refusals of the router's entry points: bad arguments end in an error on the host, before any launch."""

import ctypes

import pytest
import torch

import router_ref as R
from sgl_asap_amd import _lib
from sgl_asap_amd.moe import balance as B
from sgl_asap_amd.moe import topk as T

OK, ARG, SHAPE, UNSUP, WS = (_lib.AFD_OK, _lib.AFD_ERR_ARG, _lib.AFD_ERR_SHAPE, _lib.AFD_ERR_UNSUPPORTED,
                             _lib.AFD_ERR_WORKSPACE)


def cfg(**more):
    c = dict(num_experts=64, topk=4, scoring=0, num_groups=0, topk_groups=0, renormalize=1, scale=1.0, logits_fmt=0)
    c.update(more)
    return ctypes.byref(_lib.AfdRouterCfg(**c))


def topk(c, n=3, ld=64, logits=16, ids=16, w=16):
    return _lib.lib().afd_topk(c, logits, ld, None, None, n, ids, w, None)


@pytest.mark.parametrize("bad,status", [
    (dict(num_experts=0), SHAPE), (dict(num_experts=1025), SHAPE), (dict(topk=0), SHAPE), (dict(topk=33), SHAPE),
    (dict(num_experts=3), SHAPE), (dict(scoring=3), UNSUP), (dict(scoring=-1), UNSUP), (dict(logits_fmt=2), UNSUP),
    (dict(num_groups=-1), SHAPE), (dict(num_groups=65), SHAPE), (dict(num_groups=7, topk_groups=2), SHAPE),
    (dict(num_groups=8, topk_groups=0), SHAPE), (dict(num_groups=8, topk_groups=9), SHAPE),
    (dict(num_groups=32, topk_groups=1), SHAPE),
])
def test_bad_configs(bad, status):
    L = _lib.lib()
    assert topk(cfg(**bad)) == status
    if not set(bad) & {"num_groups", "topk_groups"}:
        assert L.afd_balance(cfg(**bad), 16, 1024, 16, None, None, 1, 3, 1.0, 16, 16, 16, 16, 1 << 30, None) == status
        assert L.afd_router_grad(cfg(**bad), 16, 1024, 16, None, 3, 16, None, 1, None, None, None, 16, None) == status
    assert L.afd_topk_balance(cfg(**bad), 16, 1024, None, None, None, 1, 3, 1.0, 16, 16, 16, 16, 16, 16, 1 << 30, None) == status


def test_bad_pointers_rows_and_workspaces():
    L = _lib.lib()
    assert topk(None) == ARG
    assert topk(cfg(), n=-1) == ARG and topk(cfg(), n=(1 << 26) + 1) == ARG
    assert topk(cfg(topk=32), n=1 << 26) == ARG  # n * topk past 31 bits
    assert topk(cfg(), ld=63) == SHAPE
    assert topk(cfg(), logits=None) == ARG and topk(cfg(), ids=None) == ARG and topk(cfg(), w=None) == ARG
    assert topk(cfg(), n=0, logits=None, ids=None, w=None) == OK
    need = ctypes.c_uint64()
    assert L.afd_balance_workspace(100, 64, 3, ctypes.byref(need)) == OK and need.value > 0
    assert L.afd_balance_workspace(-1, 64, 3, ctypes.byref(need)) == ARG
    assert L.afd_balance_workspace(100, 64, 0, ctypes.byref(need)) == ARG
    assert L.afd_balance_workspace(100, 2000, 1, ctypes.byref(need)) == SHAPE
    assert L.afd_balance_workspace(100, 64, 3, None) == ARG

    def balance(**m):
        a = dict(cfg=cfg(), logits=16, ld=64, ids=16, valid=None, cu=16, seqs=3, n=100, counts=16, coef=16, loss=16,
                 ws=16, bytes=need.value)
        a.update(m)
        return L.afd_balance(a["cfg"], a["logits"], a["ld"], a["ids"], a["valid"], a["cu"], a["seqs"], a["n"], 1.0,
                             a["counts"], a["coef"], a["loss"], a["ws"], a["bytes"], None)

    assert balance(bytes=need.value - 1) == WS and balance(ws=24) == WS
    for name in ("ids", "counts", "coef", "loss", "ws", "logits"):
        assert balance(**{name: None}) == ARG, name
    assert balance(cu=None) == ARG and balance(seqs=0) == ARG and balance(seqs=(1 << 20) + 1) == ARG

    def counts(**m):
        a = dict(ids=16, n=100, topk=4, experts=64, cu=16, seqs=3, counts=16, ws=16, bytes=need.value)
        a.update(m)
        return L.afd_expert_counts(a["ids"], a["n"], a["topk"], a["experts"], None, a["cu"], a["seqs"], a["counts"],
                                   a["ws"], a["bytes"], None)

    assert counts(bytes=need.value - 1) == WS and counts(ids=None) == ARG and counts(counts=None) == ARG
    assert counts(topk=33) == SHAPE and counts(experts=0) == SHAPE and counts(n=-1) == ARG and counts(cu=None) == ARG

    def grad(**m):
        a = dict(cfg=cfg(), logits=16, ld=64, ids=16, n=100, gw=16, cu=None, seqs=1, counts=16, coef=16, gloss=16, out=16)
        a.update(m)
        return L.afd_router_grad(a["cfg"], a["logits"], a["ld"], a["ids"], None, a["n"], a["gw"], a["cu"], a["seqs"],
                                 a["counts"], a["coef"], a["gloss"], a["out"], None)

    assert grad(out=None) == ARG and grad(ids=None) == ARG and grad(counts=None) == ARG and grad(gloss=None) == ARG
    assert grad(seqs=2) == ARG and grad(ld=10) == SHAPE and grad(n=0, out=None) == OK


def test_python_refusals():
    x = torch.zeros(4, 16)
    for call in (lambda: T.select_experts(x, 2), lambda: B.select_and_balance(x, 2, alpha=1.0),
                 lambda: B.balance_loss(x, torch.zeros(4, 2, dtype=torch.int32), alpha=1.0),
                 lambda: B.expert_counts(torch.zeros(4, 2, dtype=torch.int32), 16)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError):
        T.select_experts(x.half(), 2)
    with pytest.raises(NotImplementedError):
        T.select_experts(x, 2, scoring="relu")
    with pytest.raises(ValueError):
        T.select_experts(x, 2, num_expert_group=4)
    with pytest.raises(ValueError):
        T.select_experts(x, 2, num_expert_group=0, topk_group=1)
    with pytest.raises(NotImplementedError):
        T.TopK(2, scoring_func="relu")
    with pytest.raises(ValueError):
        T.TopK(2, use_grouped_topk=True)
    with pytest.raises(ValueError):
        T.logit_rows(torch.zeros(4))
    with pytest.raises(TypeError):
        B.balance_loss(x, torch.zeros(4, 2, dtype=torch.int64), alpha=1.0)
    with pytest.raises(ValueError):
        B.balance_loss(x, torch.zeros(3, 2, dtype=torch.int32), alpha=1.0)
    with pytest.raises(TypeError):
        T.on_device("b", torch.zeros(16, dtype=torch.float64), torch.float32, (16,), x.device)
    with pytest.raises(ValueError):
        T.on_device("b", torch.zeros(15), torch.float32, (16,), x.device)
    with pytest.raises(ValueError):
        T.on_device("b", torch.zeros(32)[::2], torch.float32, (16,), x.device)


def test_rows_that_need_no_copy():
    x = torch.zeros(6, 40)
    for t, ld in ((x, 40), (x[:, 3:23], 40), (x[::2], 80), (x[:1, :7], 7)):
        rows, stride = T.logit_rows(t)
        assert rows.data_ptr() == t.data_ptr() and stride == ld
    for t in (x.t(), x[:, ::2], x[:1].expand(5, 40), x.t()[:1]):
        rows, stride = T.logit_rows(t)
        assert rows.is_contiguous() and stride == t.shape[1] and torch.equal(rows, t)


def test_reference_gradients_against_differences():
    """The 64-bit definition's own gradient (what the kernels are compared with) against differences."""
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(6, 9, generator=g)
    ids = R.choose(R.canon(logits), 3, "sigmoid")
    gw = torch.randn(6, 3, generator=g)
    cu = [0, 2, 6]
    for scoring in R.SCORINGS:
        for renorm in (True, False):
            got = R.grads(logits, ids, scoring, renorm, 1.5, gw, 2.0, 0.3, cu)

            def value(z):
                return float((R.weights(z, ids, scoring, renorm, 1.5) * gw.double()).sum()
                             + 2.0 * R.balance(z, ids, scoring, 0.3, cu))

            for t in range(6):
                for e in range(9):
                    up, down = logits.double(), logits.double()
                    up[t, e] += 1e-5
                    down[t, e] -= 1e-5
                    assert abs((value(up) - value(down)) / 2e-5 - float(got[t, e])) < 1e-7


def test_logits_of_other_dimensions():
    for shape in ((8,), (2, 3, 8)):
        with pytest.raises(ValueError):
            T.select_experts(torch.zeros(shape), 2)
        with pytest.raises(ValueError):
            B.select_and_balance(torch.zeros(shape), 2, alpha=1.0)
        with pytest.raises(ValueError):
            B.balance_loss(torch.zeros(shape), torch.zeros(shape[0], 2, dtype=torch.int32), alpha=1.0)


BIG = (1 << 32) + 8  # the entry points' 32-bit counts hold 8 of it


def test_sizes_past_32_bits_are_refused(monkeypatch):
    """Sizes are C ints at the entry points: one past their range must not come out as another, smaller one."""
    called = []
    for m in (T, B):
        monkeypatch.setattr(m, "need_gpu", lambda *a: None)
        monkeypatch.setattr(m, "launch", lambda *a: called.append(a))
    meta = lambda *shape, dtype=torch.float32: torch.empty(*shape, dtype=dtype, device="meta")
    ids = lambda *shape: meta(*shape, dtype=torch.int32)
    for call in (
        lambda: T.select_experts(meta(BIG, 4), 2), lambda: T.select_experts(meta(2, BIG), 2),
        lambda: T.select_experts(meta(BIG, 9)[:, 2:6], 2), lambda: T.select_experts(meta(BIG, 4, dtype=torch.bfloat16), 2),
        lambda: T.select_experts(meta(2, 4), BIG), lambda: T.select_experts(meta(2, 4), 2 - (1 << 32)),
        lambda: T.select_experts(meta(2, 16), 2, num_expert_group=BIG, topk_group=4),
        lambda: T.select_experts(meta(2, 16), 2, num_expert_group=8, topk_group=BIG),
        lambda: B.select_and_balance(meta(BIG, 4), 2, alpha=1.0), lambda: B.select_and_balance(meta(2, 4), BIG, alpha=1.0),
        lambda: B.balance_loss(meta(BIG, 4), ids(BIG, 2), alpha=1.0), lambda: B.balance_loss(meta(2, 4), ids(2, BIG), alpha=1.0),
        lambda: B.balance_loss(meta(2, 4), ids(2, 2), alpha=1.0, cu_seqlens=ids(BIG)),
        lambda: B.expert_counts(ids(BIG, 2), 4), lambda: B.expert_counts(ids(2, BIG), 4), lambda: B.expert_counts(ids(2, 2), BIG),
        lambda: B.expert_counts(ids(2, 2), 4, cu_seqlens=ids(BIG)),
    ):
        with pytest.raises(ValueError, match="32 bits"):
            call()
    assert not called

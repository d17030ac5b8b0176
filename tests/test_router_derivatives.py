"""Derivatives that the router's operators and the dense FP8 layer do not have end in an error, and the ones that they have
stay connected. On the CPU, with the launches replaced by the definitions in plain torch."""

import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from sgl_asap_amd.moe import balance as B
from sgl_asap_amd.moe import linear as L
from sgl_asap_amd.moe import topk as T

TOP_K = 2


def fake_choose(cfg, top_k, logits, bias, valid):
    rows, _ = T.logit_rows(logits)
    best = torch.softmax(rows.detach(), 1).topk(top_k, 1)
    return rows, best.indices.to(torch.int32), best.values.contiguous()


def fake_grad(cfg, logits, ids, valid, gw, cu=None, counts=None, coef=None, gloss=None):
    with torch.no_grad():
        out = 3.0 * logits * logits  # any function of the logits: what is tested is what is tied to it
        if gw is not None:
            out = out + gw.sum(1, keepdim=True)
        return out.clone()


def fake_launch(name, device, *args):
    pass


@pytest.fixture
def plain(monkeypatch):
    for m in (T, B):
        for name, fake in (("need_gpu", lambda *a: None), ("router_grad", fake_grad), ("launch", fake_launch)):
            monkeypatch.setattr(m, name, fake)
    monkeypatch.setattr(T, "choose", fake_choose)
    monkeypatch.setattr(torch, "empty", torch.zeros)  # what a launch would have written


def values(which, x):
    """The differentiable outputs, one scalar whose gradient by them is a constant."""
    ids = torch.zeros(x.shape[0], TOP_K, dtype=torch.int32)
    if which == "select":
        return T.select_experts(x, TOP_K).topk_weights.sum()
    if which == "balance":
        return B.balance_loss(x, ids, alpha=1.0)[0]
    out, loss, _ = B.select_and_balance(x, TOP_K, alpha=1.0)
    return out.topk_weights.sum() + loss


ROWS = {"contiguous": lambda x: x, "strided": lambda x: x[:, 2:8], "columns": lambda x: x[:, ::2], "one row": lambda x: x[:1].expand(5, 10)}


@pytest.mark.parametrize("rows", sorted(ROWS))
@pytest.mark.parametrize("which", ["select", "balance", "both"])
def test_second_derivative_raises_whatever_it_is_mixed_with(plain, which, rows):
    leaf = torch.randn(4, 10, generator=torch.Generator().manual_seed(0)).requires_grad_()
    value = values(which, ROWS[rows](leaf))
    (g,) = torch.autograd.grad(value, leaf, create_graph=True)
    assert g.requires_grad
    # the incoming gradient was a constant, and the penalty comes with a term that has a derivative
    with pytest.raises(RuntimeError, match="no derivative of its own"):
        ((leaf ** 2).sum() + (g ** 2).sum()).backward()
    # the first derivative is the plain one
    (again,) = torch.autograd.grad(values(which, ROWS[rows](leaf)), leaf)
    assert not again.requires_grad and torch.equal(again, g.detach())


@pytest.mark.parametrize("which", ["select", "balance", "both"])
def test_a_gradient_made_with_its_graph_accumulates_like_any_other(plain, which):
    leaf = torch.ones(3, 6).requires_grad_()
    values(which, leaf).backward(create_graph=True)
    once = leaf.grad.detach().clone()
    values(which, leaf).backward(create_graph=True)
    assert torch.equal(leaf.grad.detach(), 2 * once)
    with torch.no_grad():
        leaf.grad.zero_()
    leaf.grad = None


def test_tangents_are_refused(plain, monkeypatch):
    """A dual tensor does not require a gradient, so nothing else would notice that its tangent is dropped."""
    x = torch.ones(3, 6)
    layer = object.__new__(L.Fp8BlockLinear)
    torch.nn.Module.__init__(layer)
    layer.image, layer.in_features, layer.out_features = torch.zeros(1), 6, 4
    h = torch.ones(3, 6, dtype=torch.bfloat16)
    with fw.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for t in (fw.make_dual(x, x), fw.make_dual(x, x)[:, :5], fw.make_dual(x, x)[:, ::2]):
                    for which in ("select", "balance", "both"):
                        with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                            values(which, t)
                for args in ((fw.make_dual(h, h),), (h, fw.make_dual(h[:, :4].clone(), h[:, :4].clone()))):
                    with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                        layer(*args)
                with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                    layer.silu_mul(fw.make_dual(torch.cat([h, h], 1), torch.cat([h, h], 1)))
        # no tangent, no refusal, also while a level is open
        values("select", x), values("balance", x), values("both", x)


def traced(how, f, x):
    if how == "jit":
        return torch.jit.trace(f, (x,), check_trace=False)
    return make_fx(f, tracing_mode="real", pre_dispatch=how == "pre_dispatch")(x)


@pytest.mark.parametrize("how", ["fx", "pre_dispatch", "jit"])
def test_tracing_is_refused(monkeypatch, how):
    """A trace would hold the allocation of the results and not the launch that writes them."""
    done, call = [], T._lib.call
    monkeypatch.setattr(T._lib, "call", lambda name, *args: call(name, *args) if "workspace" in name else done.append(name))
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: None)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0)
    for m in (T, B):
        monkeypatch.setattr(m, "need_gpu", lambda *a: None)
    layer = object.__new__(L.Fp8BlockLinear)
    torch.nn.Module.__init__(layer)
    layer.image, layer.in_features, layer.out_features, layer._weights_ref = torch.zeros(1), 6, 4, None
    x = torch.ones(3, 6)
    ids = torch.zeros(3, TOP_K, dtype=torch.int32)
    calls = [lambda x: T.select_experts(x, TOP_K).topk_weights, lambda x: values("balance", x), lambda x: values("both", x),
             lambda x: B.expert_counts(ids, 6), lambda x: layer(x.to(torch.bfloat16))]
    for f in calls:
        done.clear()
        f(x)
        assert len(done) == 1
        with pytest.raises(NotImplementedError, match="cannot be traced"):
            traced(how, f, x)
        # a mode that records nothing (here one that counts operations) is no trace
        with FlopCounterMode(display=False):
            f(x)
        assert len(done) == 2


def test_compiled_functions_run_the_launch_each_time(monkeypatch):
    """torch.compile breaks its graph at the call, which then runs as it is, on each call's own memory."""
    calls = []

    class Lib:
        def afd_topk(self, cfg, logits, ld, bias, valid, n, ids, w, stream):
            calls.append(n)
            ctypes.memset(ids, 0, n * TOP_K * 4)
            (ctypes.c_float * (n * TOP_K)).from_address(w)[:] = [float(len(calls))] * (n * TOP_K)
            return 0

    fake = Lib()
    monkeypatch.setattr(T._lib, "lib", lambda: fake)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: None)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0)
    monkeypatch.setattr(T, "need_gpu", lambda *a: None)

    def f(x):
        out = T.select_experts(x * 2, TOP_K)
        return out.topk_weights + 1, out.topk_ids

    torch._dynamo.reset()
    compiled = torch.compile(f, backend="eager")
    for i in range(3):
        w, ids = compiled(torch.randn(3, 6))
        assert len(calls) == i + 1 and (w == i + 2).all() and (ids == 0).all()
    torch._dynamo.reset()


@pytest.mark.parametrize("which", ["balance", "both"])
def test_counts_belong_to_the_caller(plain, monkeypatch, which):
    """What a caller does to the counts before the backward (adds them up over ranks, say: collectives write without
    autograd's notice) does not reach the gradient."""
    seen = []

    def grad(cfg, logits, ids, valid, gw, cu=None, counts=None, coef=None, gloss=None):
        seen.append(counts.clone())
        return fake_grad(cfg, logits, ids, valid, gw)

    monkeypatch.setattr(B, "router_grad", grad)
    for change in (lambda c: c.data.fill_(7), lambda c: c.add_(7)):
        leaf = torch.ones(3, 6).requires_grad_()
        if which == "both":
            _, loss, counts = B.select_and_balance(leaf, TOP_K, alpha=1.0)
        else:
            loss, counts = B.balance_loss(leaf, torch.zeros(3, TOP_K, dtype=torch.int32), alpha=1.0)
        change(counts)
        loss.backward()
        assert (counts == 7).all() and (seen.pop() == 0).all()

"""GPU: the MoE block of an attention rank as it is used: router logits -> TopK -> AsapMoE over the
one-GPU loop, with the FP8 shared expert beside the routed ones -> counts of where the tokens went; and
a training step of the router."""

import numpy as np
import pytest
import torch

import router_ref as R
from gpu_util import bits16, dev, say
from oracle import experts as OX
from sgl_asap_amd import workloads as W
from sgl_asap_amd.loop import OneGpuAfd
from sgl_asap_amd.moe import balance as B
from sgl_asap_amd.moe.experts import AfdExperts, pack_fp8_block_experts
from sgl_asap_amd.moe.layer import AsapMoE
from sgl_asap_amd.moe.shared import Fp8SharedExpertMLP
from sgl_asap_amd.moe.topk import StandardTopKOutput, TopK

pytestmark = pytest.mark.gpu

H, I, E, K = 512, 256, 32, 4
LOCAL = range(0, E)


def e4m3(shape, gen):
    return (torch.randn(*shape, generator=gen) * 60).clamp(-448, 448).to(torch.float8_e4m3fn)


def shared_expert(gen):
    blocks = lambda n, k: torch.rand(-(-n // 128), -(-k // 128), generator=gen) * 5e-4
    parts = e4m3((2 * I, H), gen), blocks(2 * I, H), e4m3((H, I), gen), blocks(H, I)
    return Fp8SharedExpertMLP(*(t.to(dev()) for t in parts))


@pytest.mark.parametrize("scoring", ["sigmoid", "sqrtsoftplus", "softmax"])
def test_block_over_the_loop(scoring):
    gen = W.generator("cpu", 3)
    w13, w2 = W.expert_weights(E, H, I, gen, "cpu")
    experts = {0: AfdExperts(E, K, 0, LOCAL, pack_fp8_block_experts(w13, w2, device=dev()), n_max=128)}
    gate = (torch.randn(E, H, generator=gen) * 0.05).to(dev())
    bias = (torch.randn(E, generator=gen) * 0.05).to(dev())
    topk = TopK(K, use_grouped_topk=True, num_expert_group=8, topk_group=4, scoring_func=scoring,
                correction_bias=bias, routed_scaling_factor=1.5)
    shared = shared_expert(gen)
    total = torch.zeros(E, dtype=torch.int64, device=dev())
    with OneGpuAfd(experts, n_max=128):
        layer = AsapMoE(E, H, I, 0, top_k=K, shared_experts=shared)
        for n, real in ((1, 1), (128, 128), (96, 61)):  # one token, a full batch, a batch padded behind 61
            say(f"block {scoring} n={n} real={real}")
            x = W.tokens(n, H, gen, "cpu").to(dev())
            valid = torch.arange(n, device=dev()) < real
            logits = x.float() @ gate.t()
            picked = topk(logits, valid)
            out = layer(x, picked)
            counts = B.expert_counts(picked.topk_ids, E)
            total += counts
            torch.cuda.synchronize()
            ids = R.choose(R.canon(logits), K, scoring, bias.cpu(), 8, 4).masked_fill(~valid.cpu()[:, None], -1)
            assert torch.equal(picked.topk_ids.cpu().long(), ids)
            assert torch.equal(counts.cpu().long(), R.counts(ids, E)[0])
            routed = experts[0](x, picked)
            torch.cuda.synchronize()
            assert np.array_equal(bits16(out), OX.combine([bits16(routed)], bits16(shared(x))))
            # a row that holds no token has no experts: the shared expert's output alone
            assert (bits16(routed)[real:] == 0).all() and (bits16(routed)[:real] != 0).any(1).all()
    assert int(total.sum()) == (1 + 128 + 61) * K


def test_block_with_bf16_logits_takes_a_strided_projection():
    """A fused projection whose last columns are the router's logits: rows with a stride."""
    gen = W.generator("cpu", 4)
    w13, w2 = W.expert_weights(E, H, I, gen, "cpu")
    experts = AfdExperts(E, K, 0, LOCAL, pack_fp8_block_experts(w13, w2, device=dev()), n_max=64)
    x = W.tokens(50, H, gen, "cpu").to(dev())
    proj = (torch.randn(H, 100 + E, generator=gen) * 0.05).to(torch.bfloat16).to(dev())
    logits = torch.mm(x, proj)[:, 100:]
    say("strided bf16 logits")
    a = experts(x, TopK(K)(logits))
    b = experts(x, TopK(K)(logits.contiguous()))
    torch.cuda.synchronize()
    assert np.array_equal(bits16(a), bits16(b)) and (bits16(a) != 0).any(1).all()


def test_training_step_of_the_router():
    """Gradient of the gate's weight from the weights' gradient and the balance loss, and bias updates
    from the counts that even the load out."""
    gen = torch.Generator().manual_seed(9)
    n, cu, alpha = 200, [0, 60, 200], 0.1
    x = torch.randn(n, H, generator=gen)
    gate = torch.randn(E, H, generator=gen) * 0.05
    gw = torch.randn(n, K, generator=gen)
    say("training step")
    leaf = gate.to(dev()).requires_grad_()
    cu_dev = torch.tensor(cu, dtype=torch.int32, device=dev())
    logits = x.to(dev()) @ leaf.t()
    out, loss, counts = B.select_and_balance(logits, K, alpha=alpha, scoring="sigmoid", cu_seqlens=cu_dev)
    ((out.topk_weights * gw.to(dev())).sum() + loss).backward()
    # the gradient at the same logits in 64 bits (the products of torch on either side are not what is tested)
    d = R.grads(logits.detach(), out.topk_ids.cpu().long(), "sigmoid", gw=gw, gl=1.0, alpha=alpha, cu=cu)
    want = d.t() @ x.double()
    mass = d.abs().t() @ x.double().abs()
    # the logits' gradient is off by 2^-16 of gw's largest (test_gpu_router), the product by n roundings
    bound = 2.0**-16 * float(gw.abs().max()) * x.double().abs().sum(0)[None] + n * 2.0**-24 * mass
    assert ((leaf.grad.cpu().double() - want).abs() <= bound).all()
    # balancing by the bias alone: each step's load is that of the choice at that step's bias
    bias = torch.zeros(E, device=dev())
    with torch.no_grad():
        for _ in range(5):
            ids = TopK(K, scoring_func="sigmoid", correction_bias=bias)(logits.detach()).topk_ids
            load = B.expert_counts(ids, E)
            chosen = R.choose(R.canon(logits.detach()), K, "sigmoid", bias.cpu())
            assert torch.equal(ids.cpu().long(), chosen)
            assert torch.equal(load.cpu().long(), R.counts(chosen, E)[0])
            bias += 0.01 * torch.sign(load.float().mean() - load)


def test_ids_and_weights_go_straight_into_the_expert_call():
    gen = W.generator("cpu", 6)
    w13, w2 = W.expert_weights(E, H, I, gen, "cpu")
    experts = AfdExperts(E, K, 0, LOCAL, pack_fp8_block_experts(w13, w2, device=dev()), n_max=64)
    x = W.tokens(33, H, gen, "cpu").to(dev())
    logits = torch.randn(33, E, generator=gen).to(dev())
    say("captured router and expert call")
    topk = TopK(K, scoring_func="sqrtsoftplus")
    want = experts(x, topk(logits)).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        experts(x, topk(logits))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = experts(x, topk(logits))
    for i in range(3):
        if i:
            logits.copy_(torch.randn(33, E, generator=gen).to(dev()))
            picked = topk(logits)
            want = experts(x, StandardTopKOutput(picked.topk_weights, picked.topk_ids)).clone()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(bits16(out), bits16(want)), i

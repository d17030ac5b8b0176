"""GPU: what the expert calls write into a caller's tensors is an in-place change to autograd."""

import pytest
import torch

from gpu_util import dev, say
from sgl_asap_amd import workloads as W
from sgl_asap_amd.moe.experts import AfdExperts, pack_fp8_block_experts, quant_act
from sgl_asap_amd.moe.topk import StandardTopKOutput
from sgl_asap_amd.runner.graph_runner import FfnGraphRunner

pytestmark = pytest.mark.gpu

H, I, E, K, N = 256, 128, 8, 2, 12


def check_saved(buf, write):
    """write() changes buf, which a product saved before."""
    w = torch.ones(H, device=dev(), dtype=torch.bfloat16, requires_grad=True)
    y = buf @ w
    write()
    with pytest.raises(RuntimeError, match="inplace operation"):
        y.sum().backward()


def test_outputs_into_a_buffer():
    gen = W.generator("cpu", 0)
    w13, w2 = W.expert_weights(E, H, I, gen, "cpu")
    experts = AfdExperts(E, K, 0, range(0, E), pack_fp8_block_experts(w13, w2, device=dev()), n_max=64)
    x = W.tokens(N, H, gen, "cpu").to(dev())
    ids, w = W.route_uniform(N, E, K, gen, "cpu")
    topk = StandardTopKOutput(w.to(dev()), ids.to(dev()))
    buf = torch.zeros(N, H, dtype=torch.bfloat16, device=dev())
    say("expert calls into a buffer")
    want = experts(x, topk)
    check_saved(buf, lambda: experts(x, topk, out=buf))
    assert torch.equal(buf, want)
    check_saved(buf, lambda: experts.forward_batch([(x, topk)], outs=[buf]))
    q, s = experts.quant_act(x)
    check_saved(buf, lambda: experts.forward_q(q, s, topk, out=buf))
    runner = FfnGraphRunner({0: experts}, 64, experts.local)
    check_saved(buf, lambda: runner.run(0, x, topk.topk_ids, topk.topk_weights, out=buf))
    check_saved(runner.run(0, x, topk.topk_ids, topk.topk_weights, 0),
                lambda: runner.run(0, -x, topk.topk_ids, topk.topk_weights, 0))
    # the runner's buffers are two tensors
    first = runner.run(0, x, topk.topk_ids, topk.topk_weights, 0)
    weight = torch.ones(H, device=dev(), dtype=torch.bfloat16, requires_grad=True)
    y = first @ weight
    runner.run(0, -x, topk.topk_ids, topk.topk_weights, 1)
    y.sum().backward()
    versions = q._version, s._version
    quant_act("fp8_1x128", x, q, s)
    assert q._version > versions[0] and s._version > versions[1]

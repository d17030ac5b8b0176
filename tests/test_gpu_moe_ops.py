"""GPU: the operators around a MoE block's experts together, as a program uses them: a training step through norm,
router, sorted tokens, experts, and norm and residual; and a decoder layer's MoE block over the one-GPU loop with an int8
shared expert."""

import numpy as np
import pytest
import torch

from gpu_util import bits16, dev, say
from oracle import experts as OX
from sgl_asap_amd import workloads as W
from sgl_asap_amd.loop import OneGpuAfd
from sgl_asap_amd.moe import balance as B
from sgl_asap_amd.moe.experts import AfdExperts, pack_fp8_block_experts
from sgl_asap_amd.moe.layer import AsapMoE
from sgl_asap_amd.moe.linear import Int8Linear
from sgl_asap_amd.moe.norm import BlockNorms, residual_norm, rms_norm
from sgl_asap_amd.moe.shared import Int8SharedExpertMLP
from sgl_asap_amd.moe.sort import sort_tokens, unsort_tokens
from sgl_asap_amd.moe.topk import TopK, select_experts

pytestmark = pytest.mark.gpu

H, I, E, K = 512, 256, 32, 4


def parameters(seed, hidden=64, inter=48, experts=6):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, scale=1.0: scale * torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    return dict(w_in=1 + 0.2 * r(hidden), w_post=1 + 0.2 * r(hidden), gate=torch.tanh(r(hidden)), w_next=1 + 0.2 * r(hidden),
                router=r(experts, hidden, scale=0.3), up=r(experts, inter, hidden, scale=0.12), down=r(experts, hidden, inter, scale=0.12))


def plain_block(x, p, ids, cfg):
    """The block in torch's own operations (64 bits), with the experts given."""
    rms = lambda v, w: v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
    normed = rms(x, p["w_in"])
    scores = torch.sigmoid(normed @ p["router"].t())
    w = scores.gather(1, ids.clamp_min(0))
    w = w / w.sum(-1, keepdim=True) * (ids >= 0)
    hidden = torch.einsum("nkih,nh->nki", p["up"][ids.clamp_min(0)], normed)
    y = torch.einsum("nkhi,nki->nkh", p["down"][ids.clamp_min(0)], torch.nn.functional.silu(hidden))
    h = x + cfg["scale"] * p["gate"] * rms((y * w[..., None]).sum(1), p["w_post"])
    return h, rms(h, p["w_next"])


def block(x, p, valid, cfg):
    """The same through the framework, in x's type."""
    normed = rms_norm(x, p["w_in"])
    topk = select_experts(normed.float() @ p["router"].t(), K, scoring="sigmoid", valid=valid)
    rows, order = sort_tokens(normed, topk.topk_ids, p["router"].shape[0])
    ends = order.offsets.tolist()
    parts = [torch.nn.functional.silu(rows[a:b] @ u.t()) @ d.t()
             for a, b, u, d in zip(ends, ends[1:], p["up"].to(x.dtype), p["down"].to(x.dtype))]
    parts.append(rows.new_zeros(rows.shape[0] - ends[-1], rows.shape[1]))
    y = unsort_tokens(torch.cat(parts), order, topk.topk_weights)
    return residual_norm(y, x, post_weight=p["w_post"], gate=p["gate"], scale=cfg["scale"], next_weight=p["w_next"]), topk, order


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_training_step(dtype):
    n, real, cfg = 150, 130, dict(scale=0.7)
    raw = parameters(5)
    g = torch.Generator().manual_seed(1)
    x0 = torch.randn(n, 64, generator=g).to(dtype)
    gh, gn = (torch.randn(n, 64, generator=g).to(dtype) for _ in range(2))
    valid = torch.arange(n, device=dev()) < real
    say(f"training step {dtype}")
    x = x0.to(dev()).requires_grad_()
    p = {k: v.float().to(dev()).requires_grad_() for k, v in raw.items()}
    out, topk, order = block(x, p, valid, cfg)
    grads = torch.autograd.grad(out, [x, *p.values()], (gh.to(dev()), gn.to(dev())))
    ids = topk.topk_ids.cpu().long()
    assert (ids[real:] == -1).all() and int(order.offsets[-1]) == real * K
    assert torch.equal(order.counts, B.expert_counts(topk.topk_ids, 6))
    xd = x0.double().requires_grad_()
    pd = {k: v.detach().cpu().double().requires_grad_() for k, v in p.items()}
    h, normed = plain_block(xd, pd, ids, cfg)
    want = torch.autograd.grad((h, normed), [xd, *pd.values()], (gh.double(), gn.double()))
    # a chain of about ten roundings of each type, none of which cancels in the norm over a tensor: 16 half steps
    tol = 16 * torch.finfo(dtype).eps / 2
    for name, got, exp in [("h", out.hidden, h), ("normed", out.normed, normed)] + list(zip(["x", *p], grads, want)):
        rel = float((got.detach().double().cpu() - exp).norm() / exp.norm())
        assert rel <= tol, (name, rel)
    # a token that is padding: its residual alone
    assert torch.equal(out.hidden[real:], x[real:])


def test_training_step_is_the_same_in_a_graph():
    n, cfg = 90, dict(scale=1.0)
    raw = parameters(6)
    x = torch.randn(n, 64, generator=torch.Generator().manual_seed(2)).to(dev())
    w = {k: v.float().to(dev()) for k, v in raw.items()}
    ids = torch.randint(0, 6, (n, K), generator=torch.Generator().manual_seed(3)).int().to(dev())
    weights = torch.rand(n, K, generator=torch.Generator().manual_seed(4)).to(dev())
    say("captured step")

    def step():
        xs, ws = x.detach().requires_grad_(), weights.detach().requires_grad_()
        p = {k: v.detach().requires_grad_() for k, v in w.items()}
        rows, order = sort_tokens(rms_norm(xs, p["w_in"]), ids, 6)
        y = unsort_tokens(rows * 2.0, order, ws)
        out = residual_norm(y, xs, post_weight=p["w_post"], gate=p["gate"], scale=cfg["scale"], next_weight=p["w_next"])
        leaves = [xs, ws, p["w_in"], p["w_post"], p["gate"], p["w_next"]]
        return [*out, *torch.autograd.grad(out, leaves, (xs.detach(), xs.detach()))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        g = torch.Generator().manual_seed(20 + i)
        x.copy_(torch.randn(n, 64, generator=g).to(dev()))
        ids.copy_(torch.randint(-1, 6, (n, K), generator=g).int().to(dev()))
        graph.replay()
        want = [t.detach().clone() for t in step()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), i


def int8(gen, rows, columns):
    return (torch.randint(-127, 128, (rows, columns), generator=gen, dtype=torch.int8).to(dev()),
            (torch.rand(rows, generator=gen) * 5e-4).to(dev()))


def test_decoder_layer_over_the_loop():
    """norms.before -> router -> AsapMoE over the loop with the int8 shared expert -> norms.after: the parts' own results,
    bit for bit."""
    gen = W.generator("cpu", 3)
    w13, w2 = W.expert_weights(E, H, I, gen, "cpu")
    experts = {0: AfdExperts(E, K, 0, range(0, E), pack_fp8_block_experts(w13, w2, device=dev()), n_max=128)}
    router = (torch.randn(E, H, generator=gen) * 0.05).to(dev())
    topk = TopK(K, scoring_func="sigmoid")
    shared = Int8SharedExpertMLP(*int8(gen, 2 * I, H), *int8(gen, H, I))
    weights = [(1 + 0.1 * torch.randn(H, generator=gen)).to(torch.bfloat16).to(dev()) for _ in range(3)]
    norms = BlockNorms(weights[0], weights[1], torch.tanh(torch.randn(H, generator=gen)).to(dev()), scale=0.5)
    with torch.no_grad(), OneGpuAfd(experts, n_max=128):
        layer = AsapMoE(E, H, I, 0, top_k=K, shared_experts=shared, norms=norms)
        for n in (1, 128, 37):
            say(f"decoder layer n={n}")
            x = W.tokens(n, H, gen, "cpu").to(dev())
            normed = layer.norms.before(x)
            picked = topk(normed.float() @ router.t())
            plain = layer(normed, picked)
            out = layer(normed, picked, residual=x, next_weight=weights[2])
            torch.cuda.synchronize()
            routed = experts[0](normed, picked)
            torch.cuda.synchronize()
            assert np.array_equal(bits16(plain), OX.combine([bits16(routed)], bits16(shared(normed))))
            want = residual_norm(plain, x, post_weight=weights[1], gate=norms.gate, scale=0.5, next_weight=weights[2])
            assert torch.equal(out.hidden, want.hidden) and torch.equal(out.normed, want.normed)
            assert torch.equal(layer(normed, picked, residual=x).hidden, want.hidden)


def test_sorted_tokens_through_int8_experts():
    """Serving: a rank's rows into its own buffer, each expert an int8 layer over its rows, and back."""
    gen = torch.Generator().manual_seed(8)
    n, hidden, experts = 60, 256, 5
    x = torch.randn(n, hidden, generator=gen).to(torch.bfloat16).to(dev())
    ids = torch.stack([torch.randperm(8, generator=gen)[:3] for _ in range(n)]).int().to(dev())
    w = torch.rand(n, 3, generator=gen).to(dev())
    layers = [Int8Linear(*int8(gen, hidden, hidden)) for _ in range(experts)]
    buffer = torch.zeros(n * 3, hidden, dtype=torch.bfloat16, device=dev())
    say("int8 experts")
    rows, order = sort_tokens(x, ids, experts, expert_lo=2, out=buffer)
    ends = order.offsets.tolist()
    back = torch.zeros_like(buffer)
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        layers[e](rows[a:b], out=back[a:b])
    out = unsort_tokens(back, order, w)
    every = torch.stack([layer(x) for layer in layers], 1).double()  # a row's result does not depend on its neighbours
    here = (ids >= 2) & (ids < 7)
    terms = every.gather(1, (ids - 2).clamp(0, 4).long()[..., None].expand(n, 3, hidden)) * (w.double() * here)[..., None]
    # three products and sums in fp32, then half a bf16 step
    bound = 2.0**-8 * terms.sum(1).abs() + 6 * 2.0**-24 * terms.abs().sum(1)
    assert ((out.double() - terms.sum(1)).abs() <= bound).all()

"""GPU: every entry of the router's gradients against its own size, in 64 bits.

Reference. With p the shares of all experts (s over their sum), q the shares of the chosen ones, r the slope ds/dl over s:

  loss:                    r_e p_e f (D_e - sum_j D_j p_j),  D = counts - counts of the row's largest share,
                           f = incoming gradient alpha E / (S' k T^2)
  weights, renormalized:   r_i q_i scale (G_i - sum_j G_j q_j),  G = g - g of the largest chosen share
  weights, softmax:        p_e scale (G_e - sum_j G_j p_j),  G = g (0 where not chosen) - g of the largest share
  weights, else:           r_i s_i scale g_i

(counting from the largest share's changes nothing in exact arithmetic and loses nothing where one share is close to one).

Tolerance, per entry, of its bound (the formula with every term positive): a share's or score's fp32 exponential is off by
|x| 2^-24 with |x| <= 40 here, its sum of up to 1024 terms (a tree of 10, 16 in a lane) and its reciprocal by less than 24 of
2^-24: 2^-18 in all. The entry takes that for its own share, again for the sum's shares, and less than it for the slope;
differences, factors and the sum's additions are below 32 of 2^-24 = 2^-19. 2^-18 (1 + 1 + 1 + 1/2) < 2^-16. Where the
logits are bf16, half a step of the entry besides (eps / 2 = 2^-8)."""

import math

import pytest
import torch

import router_ref as R
from gpu_util import dev, say
from sgl_asap_amd.moe import balance as B
from sgl_asap_amd.moe import topk as T

pytestmark = pytest.mark.gpu

REL = 2.0**-16


def slope(z, scoring):
    if scoring == "softmax":
        return torch.ones_like(z)
    if scoring == "sigmoid":
        return torch.sigmoid(-z)
    # below -30 softplus(z) = e^z and the quotient is 1/2 to 2^-43
    soft = torch.log1p(torch.exp(-z.abs())) + z.clamp(min=0.0)
    return torch.where(z < -30, torch.full_like(z, 0.5), torch.sigmoid(z) / (2 * soft))


def shares(s):
    total = s.sum(1, keepdim=True)
    return s / torch.where(total == 0, torch.ones_like(total), total)


def around(p, value):
    """(value - mean, its bound) for shares p, value counted from the largest share's."""
    d = value - value.gather(1, p.argmax(1, keepdim=True))
    return d - (p * d).sum(1, keepdim=True), d.abs() + (p * d.abs()).sum(1, keepdim=True)


def loss_grad(z, cnt, top_k, scoring, gl, alpha, cu=None, valid=None):
    n, experts = z.shape
    p = shares(R.scores(z, scoring))
    spans = R.sequences(n, cu)
    rows = [hi - lo if valid is None else int(valid[lo:hi].sum()) for lo, hi in spans]
    used = sum(r > 0 for r in rows)
    want, bound = torch.zeros(n, experts, dtype=torch.float64), torch.zeros(n, experts, dtype=torch.float64)
    for i, (lo, hi) in enumerate(spans):
        if rows[i]:
            f = gl * alpha * experts / (used * top_k * rows[i] ** 2)
            d, b = around(p[lo:hi], cnt[i].double().expand(hi - lo, experts))
            want[lo:hi], bound[lo:hi] = p[lo:hi] * f * d, p[lo:hi] * abs(f) * b
    r = slope(z, scoring)
    live = torch.ones(n, 1, dtype=torch.float64) if valid is None else valid[:, None].double()
    return want * r * live, bound * r * live


def weights_grad(z, ids, scoring, renorm, scale, gw, valid=None):
    n, experts = z.shape
    s, r, g = R.scores(z, scoring), slope(z, scoring), gw.double()
    live = torch.ones(n, 1, dtype=torch.float64) if valid is None else valid[:, None].double()
    if not renorm and scoring == "softmax":
        d, b = around(s, torch.zeros_like(s).scatter_(1, ids, g))
        return s * scale * d * live, s * scale * b * live
    q = s.gather(1, ids)
    if renorm:
        q = shares(q)
        d, b = around(q, g)
    else:
        d, b = g, g.abs()
    put = lambda v: torch.zeros(n, experts, dtype=torch.float64).scatter_(1, ids, q * scale * v) * r * live
    return put(d), put(b)


def check(got, want, bound, dtype=torch.float32):
    got = got.cpu().double()
    tol = REL * bound + (2.0**-8 * want.abs() if dtype == torch.bfloat16 else 0.0)
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol.clamp_min(1e-300)).max())


def telling(want, bound):
    """Nearly every entry is far above its tolerance, so a gradient of zeros, or of another size, fails."""
    some = bound > 0
    assert some.any() and float((want.abs() > 16 * REL * bound)[some].double().mean()) > 0.9


def on(x, dtype=None):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=dev()) if isinstance(x, list) else x.to(dev())


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("n,experts,top_k,bias,cu", [
    (7, 6, 1, False, None), (37, 60, 4, True, [2, 12, 12, 35]), (37, 128, 17, False, [0, 30, 37]), (50, 256, 8, True, None),
    (37, 500, 8, False, [0, 37]), (37, 900, 32, True, [5, 6, 30]), (6151, 60, 4, False, [2, 12, 1500, 1500, 4000]),
    (6151, 256, 8, True, [0, 700, 5000, 6151]), (3000, 160, 6, True, None)])
def test_every_entry(n, experts, top_k, bias, cu, renorm, scoring):
    scale, alpha, gl = 1.5, 0.02, 2.0
    for dtype in (torch.float32, torch.bfloat16):
        g = torch.Generator().manual_seed(n + experts)
        # popular and unpopular experts, as a router has them: counts that differ
        logits = (torch.randn(n, experts, generator=g) * 2 + torch.randn(experts, generator=g)).to(dtype)
        b = torch.randn(experts, generator=g) * 0.05 if bias else None
        gw = torch.randn(n, top_k, generator=g)
        valid = torch.rand(n, generator=g) < 0.8
        say(f"every entry n={n} E={experts} k={top_k} {scoring} renorm={renorm} {dtype}")
        leaf = logits.to(dev()).requires_grad_()
        out, loss, cnt = B.select_and_balance(leaf, top_k, alpha=alpha, scoring=scoring, renormalize=renorm, correction_bias=on(b),
                                              routed_scaling_factor=scale, cu_seqlens=on(cu), valid=on(valid))
        z, ids = R.canon(logits), out.topk_ids.cpu().long().clamp_min(0)
        parts = [weights_grad(z, ids, scoring, renorm, scale, gw, valid),
                 loss_grad(z, cnt.cpu().view(-1, experts), top_k, scoring, gl, alpha, cu, valid)]
        for take in ((0,), (1,), (0, 1)):
            outs = [(out.topk_weights, loss)[i] for i in take]
            gs = [(on(gw), torch.tensor(gl, device=dev()))[i] for i in take]
            (got,) = torch.autograd.grad(outs, (leaf,), gs, retain_graph=True)
            want, bound = sum(parts[i][0] for i in take), sum(parts[i][1] for i in take)
            # (one pick's renormalized weight is the scale: its gradient is 0)
            if take != (0,) or not renorm or top_k > 1:
                telling(want, bound)
            check(got, want, bound, dtype)


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("spans", [None, [0, 900, 900, 5000]])
def test_every_entry_for_given_ids(spans, scoring):
    """Sequences over many workgroups; ids that repeat, that are no expert's, and rows without any."""
    n, experts, top_k, alpha = 5000, 256, 8, 1.0
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(n, experts, generator=g) * 2
    ids = (torch.rand(n, top_k, generator=g) ** 2 * (experts + 2)).to(torch.int32) - 1
    say(f"given ids {scoring} {spans}")
    leaf = logits.to(dev()).requires_grad_()
    loss, cnt = B.balance_loss(leaf, ids.to(dev()), alpha=alpha, scoring=scoring, cu_seqlens=on(spans))
    (got,) = torch.autograd.grad(loss, leaf)
    want_cnt = R.counts(ids, experts, spans)
    assert torch.equal(cnt.cpu().long().view(-1, experts), want_cnt)
    want, bound = loss_grad(R.canon(logits), want_cnt, top_k, scoring, 1.0, alpha, spans)
    telling(want, bound)
    check(got, want, bound)


def peaked(n, experts, scoring, seed):
    """Rows whose largest share is 1 - eps with eps of about 1e-6 to 1e-9, at |x| <= 40 from the reference."""
    g = torch.Generator().manual_seed(seed)
    low = {"softmax": -12.0, "sigmoid": -18.0, "sqrtsoftplus": -33.0}[scoring]
    logits = low + torch.randn(n, experts, generator=g)
    logits[torch.arange(n), torch.randint(0, experts, (n,), generator=g)] = 5.0
    return logits, g


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("n,experts,top_k", [(40, 2, 1), (40, 48, 4), (33, 128, 3), (40, 200, 8), (3000, 256, 8), (20, 700, 5)])
def test_loss_gradient_of_a_share_that_holds_nearly_all(n, experts, top_k, scoring):
    """D_e - sum D_j p_j of the largest share is the small rest of the others."""
    logits, g = peaked(n, experts, scoring, experts)
    ids = (torch.rand(n, top_k, generator=g) ** 2 * experts).to(torch.int32)
    say(f"one share, loss n={n} E={experts} {scoring}")
    leaf = logits.to(dev()).requires_grad_()
    loss, cnt = B.balance_loss(leaf, ids.to(dev()), alpha=1.0, scoring=scoring)
    (got,) = torch.autograd.grad(loss, leaf)
    want, bound = loss_grad(R.canon(logits), cnt.cpu()[None], top_k, scoring, 1.0, 1.0)
    assert (shares(R.scores(R.canon(logits), scoring)).amax(1) > 1 - 1e-3).all()
    check(got, want, bound)


@pytest.mark.parametrize("experts,top_k,bias", [(2, 1, False), (48, 1, False), (64, 4, False), (200, 3, True), (256, 8, True), (700, 5, True)])
def test_softmax_weights_gradient_of_a_share_that_holds_nearly_all(experts, top_k, bias):
    """Unrenormalized softmax weights: p (1 - p) of a p close to one, whether it was chosen or (by a bias) not."""
    n, scale = 40, 1.5
    logits, g = peaked(n, experts, "softmax", experts)
    b = None
    if bias:
        b = torch.zeros(experts)
        b[: experts // 2] = 2.0  # the peak is chosen only among these
    gw = torch.randn(n, top_k, generator=g)
    say(f"one share, weights E={experts} k={top_k}")
    leaf = logits.to(dev()).requires_grad_()
    out = T.select_experts(leaf, top_k, renormalize=False, correction_bias=on(b), routed_scaling_factor=scale)
    (got,) = torch.autograd.grad(out.topk_weights, leaf, on(gw))
    ids = out.topk_ids.cpu().long()
    star = logits.argmax(1, keepdim=True)
    assert not bias or 0 < int((ids == star).any(1).sum()) < n
    check(got, *weights_grad(R.canon(logits), ids, "softmax", False, scale, gw))


@pytest.mark.parametrize("scoring", R.SCORINGS)
@pytest.mark.parametrize("experts", [1, 2, 60, 256, 600])
def test_equal_counts_have_no_loss_gradient(experts, scoring):
    """Shares add up to one, so experts that are chosen equally often leave a gradient of exactly 0."""
    n = 2 * experts
    g = torch.Generator().manual_seed(experts)
    ids = torch.arange(n).remainder(experts).to(torch.int32)[:, None]
    say(f"equal counts E={experts} {scoring}")
    leaf = (torch.randn(n, experts, generator=g) * 2).to(dev()).requires_grad_()
    loss, cnt = B.balance_loss(leaf, ids.to(dev()), alpha=1.0, scoring=scoring)
    (got,) = torch.autograd.grad(loss, leaf)
    assert (cnt == 2).all() and abs(float(loss.detach()) - 1.0) <= REL
    assert (got == 0).all()


def test_counts_past_24_bits():
    """Counts that fp32 does not tell apart: 2^24 + 2 picks of one expert, one fewer of the other."""
    top_k, half = 32, (1 << 24) // 32
    n = 2 * half
    ids = torch.zeros(n, top_k, dtype=torch.int32, device=dev())
    ids[half:] = 1
    ids[half, :2] = -1
    ids[half, 2] = 0
    say("counts past 24 bits")
    logits = torch.zeros(n, 32, device=dev())  # the C entry wants top-k experts
    logits[:, 2:] = -math.inf
    leaf = logits.requires_grad_()
    loss, cnt = B.balance_loss(leaf, ids, alpha=1.0)
    (got,) = torch.autograd.grad(loss, leaf)
    assert cnt[:3].tolist() == [(1 << 24) + 1, (1 << 24) - 3, 0]
    # p = 1/2 each: p f (D - mean D) with D_1 - D_0 = -4
    f = 32 / (top_k * float(n) ** 2)
    want = torch.tensor([0.5 * f * 2, -0.5 * f * 2], dtype=torch.float64)
    assert ((got[:, :2].cpu().double() - want).abs() <= REL * want.abs()).all() and (got[:, 2:] == 0).all()
    assert math.isfinite(float(loss.detach()))
